"""ops.block_norm and ops.block_join (csrc/block_norm.hip) against their definition and its derivatives by autograd, in fp64 on the CPU.

`terms` is each output's formula with every term replaced by its absolute value, from the fp64 quantities.  Chains: a row sum passes at most 16
additions in a lane and 10 across lanes, its root and product 3 more; x_out, h, t, dx, m, dy follow with at most 8 operations each, two of
those sums lying on the longest way (dy): 26 + 26 + 6 * 8 = 100 roundings.  Sums over rows add a rounding a row at most."""
import pytest
import torch

from .token_helpers import bound, check_close

pytestmark = pytest.mark.gpu
F, B, H = torch.float32, torch.bfloat16, torch.float16
ROUNDINGS, EPS = 100, 1e-5


def reference(x, y, post, gate, scale, nxt, gx, gh):
    """Values and gradients (fp64 autograd), and the absolute terms of each."""
    d = lambda t: None if t is None else t.detach().double().cpu()
    leaves = {k: d(v).requires_grad_() for k, v in dict(x=x, y=y, post=post, gate=gate, next=nxt).items() if v is not None}
    unit = lambda v: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    xn, out = leaves["x"], {}
    if y is not None:
        n = leaves["y"] if post is None else unit(leaves["y"]) * leaves["post"]
        xn = scale * xn + (n if gate is None else leaves["gate"] * n)
        out["x_out"] = xn
    if nxt is not None:
        out["h"] = unit(xn) * leaves["next"]
    ups = [d(dict(x_out=gx, h=gh)[k]) for k in out]
    grads = torch.autograd.grad(list(out.values()), list(leaves.values()), ups)
    out = {k: v.detach() for k, v in out.items()}
    out.update({"g_" + k: g for k, g in zip(leaves, grads)})
    # absolute terms
    a = {k: v.detach().abs() for k, v in leaves.items()}
    mean = lambda v: v.mean(-1, keepdim=True)
    over = lambda v, like: v if v.shape == like.shape else v.sum_to_size(like.shape) if v.dim() == like.dim() else v.reshape(-1, v.shape[-1]).sum(0)
    terms, one = {}, torch.ones(1, dtype=torch.float64)
    w, g = a.get("post", one), a.get("gate", one)
    xa = a["x"]
    if y is not None:
        ry = torch.rsqrt(mean(a["y"].square()) + EPS) if post is not None else one
        n = a["y"] * ry
        xa = abs(scale) * xa + g * n * w
        terms["x_out"] = xa
    t = torch.zeros_like(xa) if y is None else d(gx).abs() if gx is not None else torch.zeros_like(xa)
    if nxt is not None:
        rx = torch.rsqrt(mean(xn.detach().square()) + EPS)
        # x' carries an error of roundings * xa: relative to its own row sum it comes back through rx once more
        spread = 1 + rx * rx * mean(xa * xn.detach().abs())
        xh = xa * rx * spread
        terms["h"] = xh * a["next"]
        gha = d(gh).abs()
        t = t + rx * spread * (gha * a["next"] + xh * mean(gha * a["next"] * xh))
        terms["g_next"] = (gha * xh).reshape(-1, x.shape[-1]).sum(0)
    terms["g_x"] = (abs(scale) if y is not None else 1.0) * t
    if y is not None:
        m = t * g * w
        terms["g_y"] = ry * (m + n * mean(m * n)) if post is not None else m
        if post is not None:
            terms["g_post"] = (t * g * n).reshape(-1, x.shape[-1]).sum(0)
        if gate is not None:
            terms["g_gate"] = over((t * n * w).expand(x.shape), a["gate"])
    return out, terms


def rows_of(shape):
    n = 1
    for s in shape[:-1]:
        n *= s
    return n


def run_join(ops, x, y, post, gate, scale, nxt, gx, gh):
    got = ops.block_join(x, y, post_weight=post, gate=gate, residual_scale=scale, next_weight=nxt, eps=EPS)
    res = dict(zip(("x_out", "h"), got if nxt is not None else (got,)))
    leaves = {k: v for k, v in dict(x=x, y=y, post=post, gate=gate, next=nxt).items() if v is not None}
    ups = [dict(x_out=gx, h=gh)[k] for k in res]
    grads = torch.autograd.grad(list(res.values()), list(leaves.values()), ups)
    res.update({"g_" + k: g for k, g in zip(leaves, grads)})
    return res


def compare(got, want, terms, rows):
    for k, v in got.items():
        assert v.dtype in (F, B, H)
        extra = rows if k in ("g_post", "g_next", "g_gate") else 0
        check_close(v, want[k], bound(want[k], v.dtype, terms[k], ROUNDINGS + extra), k)


def inputs(shape, act, stream, weights, gate_kind, post, nxt, seed):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    D = shape[-1]
    x, y = (r(*shape) * 1.5).to(stream).cuda(), (r(*shape) * 3).to(act).cuda()
    w = lambda on: (1 + 0.2 * r(D)).to(weights).cuda() if on else None
    gshape = {"none": None, "channel": (D,), "sample": (shape[0],) + (1,) * (len(shape) - 2) + (D,), "token": tuple(shape[:-1]) + (1,), "full": tuple(shape)}[gate_kind]
    gate = None if gshape is None else (0.7 * r(*gshape)).to(act if gate_kind == "full" else weights).cuda()
    gx, gh = r(*shape).to(stream).cuda(), r(*shape).to(act).cuda()
    post_w, next_w = w(post), w(nxt)
    for t in (x, y, post_w, gate, next_w):
        if t is not None:
            t.requires_grad_()
    return x, y, post_w, gate, next_w, gx, gh


JOIN = [
    # shape, act, stream, weights, gate, post, next
    ((1, 1, 8), F, F, F, "channel", True, True), ((1, 1, 1), F, F, F, "none", True, True), ((2, 3, 64), B, B, B, "sample", True, True),
    ((2, 5, 65), B, F, F, "token", True, True), ((3, 7, 128), H, H, F, "full", True, True), ((4, 33, 256), B, B, F, "channel", True, True),
    ((2, 100, 333), H, F, H, "sample", True, True), ((3, 50, 512), F, F, F, "token", True, True), ((2, 77, 520), B, B, F, "full", True, True),
    ((2, 129, 1024), B, F, F, "none", True, True), ((2, 65, 1021), B, B, B, "channel", True, False), ((1, 40, 2048), H, H, H, "sample", False, True),
    ((2, 31, 4096), B, B, F, "channel", True, True), ((1, 9, 4100), B, F, F, "token", True, True), ((1, 5, 8192), F, F, F, "full", True, True),
    ((1, 6, 9001), B, B, F, "sample", True, True), ((1, 3, 16384), B, F, F, "channel", True, True), ((1, 3, 16383), F, F, F, "full", True, True),
    ((5, 1, 700), B, B, F, "sample", True, True), ((2, 400, 72), F, F, F, "token", False, True), ((2, 30, 48), F, F, F, "none", False, False),
    ((2, 30, 48), B, B, B, "full", False, False), ((3, 4, 5, 40), F, F, F, "sample", True, True), ((1500, 1, 16), F, F, F, "sample", True, True),
]


@pytest.mark.parametrize("shape,act,stream,weights,gate,post,nxt", JOIN)
def test_join_and_its_gradients(cuda, shape, act, stream, weights, gate, post, nxt):
    from omnihd_amd import ops
    x, y, pw, g, nw, gx, gh = inputs(shape, act, stream, weights, gate, post, nxt, sum(shape))
    scale = 0.75
    got = run_join(ops, x, y, pw, g, scale, nw, gx, gh)
    want, terms = reference(x, y, pw, g, scale, nw, gx, gh)
    compare(got, want, terms, rows_of(shape))
    assert got["x_out"].dtype == stream and (not nxt or got["h"].dtype == act)
    again = run_join(ops, x, y, pw, g, scale, nw, gx, gh)
    assert all(torch.equal(got[k], again[k]) for k in got)
    with torch.no_grad():                                  # the serving form: the same values
        plain = ops.block_join(x, y, post_weight=pw, gate=g, residual_scale=scale, next_weight=nw, eps=EPS)
    plain = plain if nxt else (plain,)
    assert all(torch.equal(a, got[k]) for a, k in zip(plain, ("x_out", "h")))


@pytest.mark.parametrize("shape,x_t,out_t,weights", [((1, 8), F, F, F), ((3, 100, 256), H, H, F), ((2, 9, 1000), F, B, F), ((5, 4096), B, B, B), ((2, 16384), F, H, H),
                                                     ((70, 11), B, B, F), ((1, 12345), F, F, F), ((4000, 24), F, F, F), ((7,), F, F, F)])
def test_norm_and_its_gradients(cuda, shape, x_t, out_t, weights):
    from omnihd_amd import ops
    gen = torch.Generator().manual_seed(sum(shape))
    x = (2 * torch.randn(*shape, generator=gen)).to(x_t).cuda().requires_grad_()
    w = (1 + 0.3 * torch.randn(shape[-1], generator=gen)).to(weights).cuda().requires_grad_()
    gh = torch.randn(*shape, generator=gen).to(out_t).cuda()
    h = ops.block_norm(x, w, eps=EPS, out_dtype=out_t)
    g_x, g_next = torch.autograd.grad(h, (x, w), gh)
    want, terms = reference(x, None, None, None, 1.0, w, None, gh)
    compare({"h": h, "g_x": g_x, "g_next": g_next}, want, terms, rows_of(shape))
    assert torch.equal(ops.block_norm(x.detach(), w.detach(), eps=EPS, out_dtype=out_t), h)


@pytest.mark.parametrize("wanted", ["x", "y", "post", "gate", "next"])
@pytest.mark.parametrize("gate", ["channel", "token", "full"])
def test_single_gradients_and_missing_upstreams(cuda, wanted, gate):
    """Each gradient alone is the one of the whole; with one output unused its upstream counts as zero."""
    from omnihd_amd import ops
    x, y, pw, g, nw, gx, gh = inputs((2, 37, 200), F, F, F, gate, True, True, 5)
    whole = run_join(ops, x, y, pw, g, 0.5, nw, gx, gh)
    named = dict(x=x, y=y, post=pw, gate=g, next=nw)
    call = lambda m: ops.block_join(m["x"], m["y"], post_weight=m["post"], gate=m["gate"], residual_scale=0.5, next_weight=m["next"], eps=EPS)
    alone = {k: v.detach().requires_grad_(k == wanted) for k, v in named.items()}
    assert torch.equal(torch.autograd.grad(call(alone), alone[wanted], (gx, gh))[0], whole["g_" + wanted])
    for only in ("x_out", "h"):
        if wanted == "next" and only == "x_out":
            continue
        out = dict(zip(("x_out", "h"), call(named)))[only]
        up = dict(x_out=gx, h=gh)[only]
        got, = torch.autograd.grad(out, named[wanted], up)
        zero = dict(x_out=(gx, torch.zeros_like(gh)), h=(torch.zeros_like(gx), gh))[only]
        ref, = torch.autograd.grad(call(named), named[wanted], zero)
        assert torch.equal(got, ref)


def test_differences(cuda):
    """Directional derivatives by central differences of the operator itself, fp32 rows.  With a step s in a direction of unit values the
    quotient is off by s^2 / 6 of a third derivative (values of order 1 to 10 here: 2e-6 at s = 1e-3... 1e-2) and by the rounding of the sums,
    2^-24 * sum|terms| / s; both stay under 1e-3 of the sum of the products' absolute values."""
    from omnihd_amd import ops
    x, y, pw, g, nw, gx, gh = inputs((2, 9, 40), F, F, F, "sample", True, True, 11)
    named = dict(x=x, y=y, post=pw, gate=g, next=nw)

    def value(m):
        out, h = ops.block_join(m["x"], m["y"], post_weight=m["post"], gate=m["gate"], residual_scale=0.8, next_weight=m["next"], eps=EPS)
        return (out.double() * gx.double()).sum() + (h.double() * gh.double()).sum()
    grads = run_join(ops, x, y, pw, g, 0.8, nw, gx, gh)
    gen = torch.Generator().manual_seed(1)
    for k, v in named.items():
        step = 1e-2
        way = torch.randn(v.shape, generator=gen).cuda()
        with torch.no_grad():
            up, down = value({**named, k: v + step * way}), value({**named, k: v - step * way})
        quotient = ((up - down) / (2 * step)).item()
        products = grads["g_" + k].double() * way.double()
        assert abs(quotient - products.sum().item()) <= 2e-3 * products.abs().sum().item(), k


def test_strides_and_offsets(cuda):
    from omnihd_amd import ops
    gen = torch.Generator().manual_seed(2)
    D = 96
    store = torch.randn(50, 2 * D + 3, generator=gen).bfloat16().cuda()
    for a, b in ((slice(0, D), slice(D, 2 * D)), (slice(1, D + 1), slice(D + 3, 2 * D + 3))):
        x, y = store[:, a].detach().requires_grad_(), store[:, b].detach().requires_grad_()
        pw, nw = (torch.randn(D + 1, generator=gen).cuda()[1:].requires_grad_() for _ in range(2))
        gate = store[:, 5:5 + D].detach().requires_grad_()
        gx, gh = store[:, 7:7 + D], torch.ones(1, 1, device="cuda", dtype=B).expand(50, D)
        got = run_join(ops, x, y, pw, gate, 1.0, nw, gx, gh)
        want, terms = reference(x, y, pw, gate, 1.0, nw, gx, gh)
        compare(got, want, terms, 50)
    x = torch.randn(6, D, 5, generator=gen).cuda().transpose(1, 2).requires_grad_()          # no dense rows: copied
    h = ops.block_norm(x, nw.detach())
    assert torch.equal(h, ops.block_norm(x.detach().contiguous(), nw.detach()))


def test_no_rows(cuda):
    from omnihd_amd import ops
    x, y, pw, g, nw, gx, gh = inputs((2, 0, 40), B, F, F, "sample", True, True, 1)
    got = run_join(ops, x, y, pw, g, 1.0, nw, gx, gh)
    assert got["x_out"].shape == (2, 0, 40) and got["g_x"].shape == (2, 0, 40)
    for k in ("g_post", "g_gate", "g_next"):
        assert not got[k].any()


def test_rows_do_not_touch_one_another(cuda):
    """A row of NaN or infinities stays its own affair (its weights' gradients aside)."""
    from omnihd_amd import ops
    x, y, pw, g, nw, _, _ = inputs((1, 40, 300), B, B, F, "channel", True, True, 4)
    clean = ops.block_join(x, y, post_weight=pw, gate=g, next_weight=nw)
    bad = x.detach().clone()
    bad[0, 13], bad[0, 20] = float("nan"), float("inf")
    dirty = ops.block_join(bad, y.detach(), post_weight=pw.detach(), gate=g.detach(), next_weight=nw.detach())
    rest = [i for i in range(40) if i not in (13, 20)]
    for a, b in zip(clean, dirty):
        assert torch.equal(a[0, rest], b[0, rest]) and bool(b[0, 13].isnan().all())


def test_stream_and_graph(cuda):
    from omnihd_amd import ops
    x, y, pw, g, nw, gx, gh = inputs((2, 300, 264), B, B, F, "sample", True, True, 8)
    gen = torch.Generator().manual_seed(12)
    step = lambda: run_join(ops, x, y, pw, g, 0.9, nw, gx, gh)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        with torch.no_grad():
            for t in (x, y, gx, gh):
                t.copy_(torch.randn(t.shape, generator=gen).to(t.dtype).cuda())
        graph.replay()
        torch.cuda.synchronize()
        now = step()
        assert all(torch.equal(now[n], held[n]) for n in now), k


@pytest.mark.parametrize("missing", [("gate",), ("post",), ("post", "gate"), ("next",), ("gate", "next"), ("post", "gate", "next")])
def test_single_gradients_with_missing_weights(cuda, missing):
    """One gradient wanted, some of the weights not given: it is the one of the whole."""
    from omnihd_amd import ops
    x, y, pw, g, nw, gx, gh = inputs((3, 11, 88), F, F, F, "sample", True, True, 6)
    named = {k: None if k in missing else v for k, v in dict(x=x, y=y, post=pw, gate=g, next=nw).items()}
    whole = run_join(ops, named["x"], named["y"], named["post"], named["gate"], 0.5, named["next"], gx, gh)
    for wanted in (k for k, v in named.items() if v is not None):
        alone = {k: None if v is None else v.detach().requires_grad_(k == wanted) for k, v in named.items()}
        out = ops.block_join(alone["x"], alone["y"], post_weight=alone["post"], gate=alone["gate"], residual_scale=0.5, next_weight=alone["next"], eps=EPS)
        got, = torch.autograd.grad(out, alone[wanted], (gx, gh) if "next" not in missing else gx)
        assert torch.equal(got, whole["g_" + wanted]), wanted


def test_a_row_without_leading_dimensions(cuda):
    from omnihd_amd import ops
    x, y, pw, g, nw, gx, gh = (t[0] if t is not None and t.dim() > 1 else t for t in inputs((1, 50), B, B, F, "channel", True, True, 3))
    a = run_join(ops, *(t.detach().requires_grad_() for t in (x, y)), pw, g, 1.0, nw, gx, gh)
    x2, y2 = x.detach()[None].requires_grad_(), y.detach()[None].requires_grad_()
    b = run_join(ops, x2, y2, pw, g, 1.0, nw, gx[None], gh[None])
    for k in a:
        assert torch.equal(a[k], b[k].reshape(a[k].shape)), k


def test_offsets_beyond_32_bits(cuda):
    """More than 2^31 elements: the last rows are what they are alone."""
    from omnihd_amd import ops
    D = 4096
    rows = 2 ** 31 // D + 40
    x, y = torch.zeros(rows, D, dtype=B, device="cuda"), torch.zeros(rows, D, dtype=B, device="cuda")
    gen = torch.Generator().manual_seed(1)
    for t in (x, y):
        t[-50:] = torch.randn(50, D, generator=gen).bfloat16().cuda()
    w = torch.randn(D, generator=gen).cuda()
    gate = torch.randn(rows, 1, generator=gen).cuda()
    up = torch.zeros(rows, D, dtype=B, device="cuda")
    up[-50:] = torch.randn(50, D, generator=gen).bfloat16().cuda()
    xs, ys, ws = x[-50:].clone().requires_grad_(), y[-50:].clone().requires_grad_(), w.clone().requires_grad_()
    small = ops.block_join(xs, ys, post_weight=ws, gate=gate[-50:], next_weight=ws)
    small_g = torch.autograd.grad(small, (xs, ys), (up[-50:], up[-50:]))
    x.requires_grad_(), y.requires_grad_()
    big = ops.block_join(x, y, post_weight=w, gate=gate, next_weight=w)
    big_g = torch.autograd.grad(big, (x, y), (up, up))
    for a, b in zip((*big, *big_g), (*small, *small_g)):
        assert torch.equal(a[-50:], b) and not a[1000:1010].any()
