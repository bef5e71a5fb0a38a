"""ops.token_embedding (csrc/token_embed.hip) against its definition: the lookup bit for bit (one fp32 product, one rounding), the table's
gradient against fp64 sums.  A gradient row of c tokens is a sum of c terms in fp32 (each term exact in fp32: c - 1 roundings at
most), times the scale (1), rounded to the table's type."""
import pytest
import torch

from .token_helpers import bound, check_close

pytestmark = pytest.mark.gpu
F, B, H = torch.float32, torch.bfloat16, torch.float16


def make_ids(kind, n, vocab, gen):
    if kind == "random":
        return torch.randint(0, vocab, (n,), generator=gen)
    if kind == "same":
        return torch.full((n,), vocab // 2)
    if kind == "order":
        return torch.arange(n) % vocab
    if kind == "runs":                                     # runs of 37: they cross the borders of chunks of any size
        return (torch.arange(n) // 37) % vocab
    assert kind == "hot"                                   # half of the tokens are one and the same
    ids = torch.randint(0, vocab, (n,), generator=gen)
    ids[torch.rand(n, generator=gen) < 0.5] = vocab - 1
    return ids


def reference_grad(ids, g, vocab, scale, padding):
    """Value and sum of absolute terms, fp64."""
    ids, g = ids.reshape(-1).long().cpu(), g.detach().double().cpu().reshape(ids.numel(), -1)
    keep = (ids >= 0) & (ids < vocab)
    if padding is not None:
        keep &= ids != padding
    out, terms = (torch.zeros(vocab, g.shape[1], dtype=torch.float64) for _ in range(2))
    out.index_add_(0, ids[keep], g[keep])
    terms.index_add_(0, ids[keep], g[keep].abs())
    count = torch.zeros(vocab, dtype=torch.float64).index_add_(0, ids[keep], torch.ones(int(keep.sum()), dtype=torch.float64))
    return out * scale, terms * abs(scale), count[:, None]


CASES = [
    # n, vocab, dim, table, out, kind
    (1, 1, 1, F, F, "random"), (1, 32000, 256, B, B, "random"), (7, 5, 8, H, H, "random"), (64, 300, 64, F, B, "random"),
    (65, 1000, 33, B, B, "order"), (1000, 50, 128, F, H, "hot"), (4100, 230000, 24, F, F, "random"), (5003, 997, 333, F, B, "runs"),
    (20011, 500, 520, B, B, "hot"), (33000, 3, 72, H, H, "same"), (9000, 20000, 1024, F, B, "order"), (777, 129, 4100, B, B, "runs"),
    (2048, 4000, 7, H, H, "hot"), (513, 600, 16, F, F, "same"), (40000, 100, 40, F, F, "runs"),
    (131072, 5000, 16, F, F, "hot"), (147456, 3, 8, F, F, "random"), (150003, 200003, 8, F, B, "random"), (147455, 900, 9, F, F, "runs"), (200000, 700, 12, B, B, "same"),
    (148500, 2100000, 2, F, F, "random"), (160000, 5000, 16, B, B, "hot"), (150000, 900, 9, F, F, "runs"), (300000, 40000, 8, F, F, "order"),
]


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("n,vocab,dim,table_t,out_t,kind", CASES)
def test_lookup_and_gradient(cuda, n, vocab, dim, table_t, out_t, kind, wide):
    gen = torch.Generator().manual_seed(n + dim)
    from omnihd_amd import ops
    ids = make_ids(kind, n, vocab, gen).to(torch.int64 if wide else torch.int32)
    table = torch.randn(vocab, dim, generator=gen).to(table_t).cuda().requires_grad_()
    scale, padding = 0.37, int(ids[n // 2]) if kind == "random" and n > 7 else None
    out = ops.token_embedding(ids.cuda(), table, scale=scale, padding_idx=padding, out_dtype=out_t)
    assert out.shape == (n, dim) and out.dtype == out_t
    assert torch.equal(out, (table.detach().float() * scale).to(out_t)[ids.cuda().long()])
    assert torch.equal(ops.token_embedding(ids.cuda(), table.detach(), scale=scale, out_dtype=out_t), out)
    g = torch.randn(n, dim, generator=gen).to(out_t).cuda()
    grad, = torch.autograd.grad(out, table, g, retain_graph=True)
    assert grad.dtype == table_t and grad.is_contiguous()
    s = torch.tensor(scale, dtype=torch.float32).double().item()
    want, terms, count = reference_grad(ids, g, vocab, s, padding)
    check_close(grad, want, bound(want, table_t, terms, count + 1), "grad")
    again, = torch.autograd.grad(out, table, g)
    assert torch.equal(grad, again)


def test_ids_of_any_shape_and_outside_the_table(cuda):
    from omnihd_amd import ops
    gen = torch.Generator().manual_seed(3)
    table = torch.randn(50, 20, generator=gen).cuda().requires_grad_()
    ids = torch.randint(0, 50, (3, 4, 5), generator=gen)
    ids[0, 0, 0], ids[1, 2, 3], ids[2, 3, 4] = -1, 50, 2 ** 40
    out = ops.token_embedding(ids.cuda(), table)
    bad = (ids < 0) | (ids >= 50)
    assert out.shape == (3, 4, 5, 20) and bool(out[bad.cuda()].isnan().all()) and torch.equal(out[~bad.cuda()], table[ids[~bad].cuda()])
    g = torch.randn(3, 4, 5, 20, generator=gen).cuda()
    grad, = torch.autograd.grad(out, table, g)
    want, terms, count = reference_grad(ids, g, 50, 1.0, None)
    check_close(grad, want, bound(want, F, terms, count + 1), "grad")
    assert ops.token_embedding(ids.cuda()[:, ::2], table.detach()).shape == (3, 2, 5, 20)      # ids with strides


def test_no_tokens(cuda):
    from omnihd_amd import ops
    table = torch.randn(1000, 48, device="cuda").requires_grad_()
    ids = torch.zeros(2, 0, dtype=torch.int64, device="cuda")
    out = ops.token_embedding(ids, table)
    assert out.shape == (2, 0, 48)
    grad, = torch.autograd.grad(out.sum() if out.numel() else out.sum(), table)
    assert not grad.any()


@pytest.mark.parametrize("dim,pitch,offset", [(64, 72, 0), (64, 67, 3), (40, 40, 1), (33, 50, 8)])
def test_tables_and_gradients_with_pitch_and_offset(cuda, dim, pitch, offset):
    from omnihd_amd import ops
    gen = torch.Generator().manual_seed(dim + pitch)
    vocab, n = 210, 1500
    store = torch.randn(vocab * pitch + offset, generator=gen).bfloat16().cuda()
    table = store[offset:].view(vocab, pitch)[:, :dim].detach().requires_grad_()
    ids = torch.randint(0, vocab, (n,), generator=gen).cuda()
    out = ops.token_embedding(ids, table, scale=2.0)
    assert torch.equal(out, table.detach()[ids] * 2)
    wide = torch.randn(n, 2 * dim + 1, generator=gen).bfloat16().cuda()
    for g in (wide[:, :dim], wide[:, 1:dim + 1], wide[:, ::2][:, :dim], torch.ones(1, 1, device="cuda", dtype=B).expand(n, dim)):
        grad, = torch.autograd.grad(out, table, g, retain_graph=True)
        want, terms, count = reference_grad(ids, g, vocab, 2.0, None)
        check_close(grad, want, bound(want, B, terms, count + 1), "grad")


def test_stream_and_graph(cuda):
    """On a stream of its own, and captured: replays follow the inputs' contents, with eager work between them."""
    from omnihd_amd import ops
    gen = torch.Generator().manual_seed(9)
    vocab, n, dim = 3000, 5000, 96
    table = torch.randn(vocab, dim, generator=gen).cuda().requires_grad_()
    ids, g = torch.randint(0, vocab, (n,), generator=gen).cuda(), torch.randn(n, dim, generator=gen).cuda()

    def step():
        out = ops.token_embedding(ids, table, scale=3.0, padding_idx=7)
        return out.detach(), torch.autograd.grad(out, table, g)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out_g, grad_g = step()
    for k in range(4):
        ids.copy_(torch.randint(0, vocab, (n,), generator=gen).cuda() if k != 2 else torch.full((n,), 5).cuda())
        g.copy_(torch.randn(n, dim, generator=gen).cuda())
        graph.replay()
        torch.cuda.synchronize()
        out, grad = step()
        assert torch.equal(out, out_g) and torch.equal(grad, grad_g), k


def test_offsets_beyond_32_bits(cuda):
    """A table of more than 2^31 elements: rows at its end are looked up and get their gradient, every other row is zero."""
    from omnihd_amd import ops
    dim = 4096
    vocab = 2 ** 31 // dim + 100
    table = torch.zeros(vocab, dim, dtype=H, device="cuda")
    gen = torch.Generator().manual_seed(2)
    table[-90:] = torch.randn(90, dim, generator=gen).half().cuda()
    table.requires_grad_()
    ids = torch.tensor([vocab - 1, vocab - 90, 5, vocab - 1, vocab - 30], device="cuda")
    out = ops.token_embedding(ids, table)
    assert torch.equal(out, table.detach()[ids])
    g = torch.randn(5, dim, generator=gen).half().cuda()
    grad, = torch.autograd.grad(out, table, g)
    assert torch.equal(grad[vocab - 1], (g[0].float() + g[3].float()).half())
    assert torch.equal(grad[[vocab - 90, 5, vocab - 30]], g[[1, 2, 4]])
    grad[[vocab - 1, vocab - 90, 5, vocab - 30]] = 0
    assert all(not part.any() for part in grad.split(65536))
