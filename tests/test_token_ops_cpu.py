"""What the token operators refuse, without a GPU: the wrappers' checks (on CPU tensors that claim to be on the device; no call gets as far as
the library), and the C entry points' own."""
import ctypes

import pytest
import torch


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on the GPU: the wrappers' argument checks run on it."""
    is_cuda = True


def dev(t):
    return t.as_subclass(OnDevice)


@pytest.fixture()
def ops(monkeypatch):
    from omnihd_amd import ops
    from omnihd_amd.ops import misc, norm

    def never():
        raise AssertionError("the library was reached")
    monkeypatch.setattr(misc, "torch_ops", never)
    monkeypatch.setattr(norm, "torch_ops", never)
    return ops


def test_cpu_tensors_are_refused(ops):
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.token_embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.block_norm(torch.zeros(3, 8), torch.ones(8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.block_join(torch.zeros(3, 8), torch.zeros(3, 8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.topk_distill_loss(torch.zeros(3, 8), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64))


def test_embedding_refusals(ops):
    ids, table = dev(torch.zeros(3, dtype=torch.int64)), dev(torch.zeros(4, 8))
    for bad, error in ((dict(ids=dev(torch.zeros(3))), TypeError), (dict(ids=dev(torch.zeros(3, dtype=torch.int16))), TypeError),
                       (dict(table=dev(torch.zeros(4, 8, dtype=torch.float64))), TypeError), (dict(table=dev(torch.zeros(8))), ValueError),
                       (dict(table=dev(torch.zeros(0, 8))), ValueError), (dict(table=dev(torch.zeros(8, 4).t())), ValueError),
                       (dict(table=dev(torch.zeros(1, 8).expand(4, 8))), ValueError), (dict(padding_idx=4), ValueError), (dict(padding_idx=-5), ValueError),
                       (dict(out_dtype=torch.float64), TypeError), (dict(table=dev(torch.zeros(4, 8).bfloat16()), out_dtype=torch.float32), TypeError)):
        with pytest.raises(error):
            ops.token_embedding(**{**dict(ids=ids, table=table), **bad})


def test_norm_refusals(ops):
    x, w = dev(torch.zeros(3, 8)), dev(torch.ones(8))
    for bad, error in ((dict(weight=None), TypeError), (dict(weight=dev(torch.ones(7))), ValueError), (dict(weight=dev(torch.ones(8, 1))), ValueError),
                       (dict(eps=0.0), ValueError), (dict(eps=float("nan")), ValueError), (dict(out_dtype=torch.float64), TypeError),
                       (dict(x=dev(torch.zeros(3, 8).half()), out_dtype=torch.float32), TypeError), (dict(x=dev(torch.zeros(3, 8).double())), TypeError),
                       (dict(x=dev(torch.zeros(2, 16385)), weight=dev(torch.ones(16385))), ValueError), (dict(x=dev(torch.zeros(3, 0)), weight=dev(torch.ones(0))), ValueError)):
        with pytest.raises(error):
            ops.block_norm(**{**dict(x=x, weight=w), **bad})
    y = dev(torch.zeros(3, 8))
    for bad, error in ((dict(y=dev(torch.zeros(2, 8))), ValueError), (dict(y=dev(torch.zeros(3, 8).bfloat16()), x=dev(torch.zeros(3, 8).half())), TypeError),
                       (dict(x=dev(torch.zeros(3, 8).bfloat16())), TypeError), (dict(gate=dev(torch.zeros(7))), ValueError), (dict(gate=dev(torch.zeros(2, 8))), ValueError),
                       (dict(gate=dev(torch.zeros(1))), ValueError), (dict(post_weight=dev(torch.ones(7))), ValueError), (dict(next_weight=torch.ones(8)), RuntimeError)):
        with pytest.raises(error):
            ops.block_join(**{**dict(x=x, y=y), **bad})


@pytest.mark.parametrize("gate,rows,want", [((6,), (2, 3, 4, 6), (1, 24)), ((2, 1, 1, 6), (2, 3, 4, 6), (1, 12)), ((2, 3, 1, 6), (2, 3, 4, 6), (1, 4)),
                                            ((1, 1, 1, 6), (2, 3, 4, 6), (1, 24)), ((2, 3, 4, 6), (2, 3, 4, 6), (3, 1)), ((2, 3, 4, 1), (2, 3, 4, 6), (2, 1)),
                                            ((5, 6), (5, 6), (3, 1)), ((1, 6), (5, 6), (1, 5)), ((5, 1), (5, 6), (2, 1)), ((6,), (6,), (1, 1))])
def test_gate_layouts(ops, gate, rows, want):
    assert ops._gate_layout(torch.zeros(gate), rows) == want


@pytest.mark.parametrize("gate,rows", [((1, 3, 1, 6), (2, 3, 4, 6)), ((3, 4, 6), (2, 3, 4, 6)), ((2, 1, 4, 6), (2, 3, 4, 6)), ((4, 1), (2, 4, 6)), ((), (2, 6))])
def test_gates_that_fit_no_layout(ops, gate, rows):
    with pytest.raises(ValueError):
        ops._gate_layout(torch.zeros(gate), rows)


def test_distill_refusals(ops):
    good = dict(logits=dev(torch.zeros(3, 8)), teacher_logits=dev(torch.zeros(3, 2)), teacher_ids=dev(torch.zeros(3, 2, dtype=torch.int64)))
    wide = dict(teacher_logits=dev(torch.zeros(3, 257)), teacher_ids=dev(torch.zeros(3, 257, dtype=torch.int64)))
    none = dict(teacher_logits=dev(torch.zeros(3, 0)), teacher_ids=dev(torch.zeros(3, 0, dtype=torch.int64)))
    for bad, error in ((dict(logits=dev(torch.zeros(3, 8).double())), TypeError), (dict(logits=dev(torch.zeros(3, 0))), ValueError), (dict(teacher_ids=dev(torch.zeros(3, 2))), TypeError),
                       (dict(teacher_ids=dev(torch.zeros(3, 3, dtype=torch.int64))), ValueError), (dict(logits=dev(torch.zeros(4, 8))), ValueError), (wide, ValueError), (none, ValueError),
                       (dict(temperature=0.0), ValueError), (dict(temperature=float("nan")), ValueError), (dict(temperature=-1.0), ValueError), (dict(reduction="batchmean"), ValueError),
                       (dict(reduction="sum", avg_factor=3.0), ValueError), (dict(row_weight=dev(torch.ones(4))), ValueError), (dict(row_weight=[1, 1, 1]), ValueError),
                       (dict(avg_factor=dev(torch.ones(2))), ValueError)):
        with pytest.raises(error):
            ops.topk_distill_loss(**{**good, **bad})


def test_c_entries_refuse_before_any_launch():
    """Bad sizes, types, null pointers and short workspaces come back as a status with a text; nothing is launched (there is no GPU here)."""
    from omnihd_amd._lib import lib
    L = lib()
    p = ctypes.c_void_p(64)                                # never read: every call below is refused first
    ARG, WORKSPACE = -1, -3
    embed = [p, 1, 5, p, 0, 8, 4, 8, 1.0, p, 0, None]
    for at, bad in ((2, -1), (2, 1 << 31), (6, 0), (6, 1 << 31), (7, 0), (7, (1 << 24) + 1), (4, 3), (10, 2 + 5), (4, 1), (5, 7), (0, None), (3, None), (9, None)):
        args = list(embed)
        args[at] = bad
        assert L.omnihd_token_embed_fwd(*args) == ARG, (at, bad)
        assert L.omnihd_last_error()
    need = L.omnihd_token_embed_bwd_workspace_bytes(5, 7, 8)
    back = [p, 1, 5, p, 0, 8, 7, 8, 1.0, -1, p, 0, p, need, None]
    for at, bad, status in ((13, need - 1, WORKSPACE), (12, None, ARG), (10, None, ARG), (3, None, ARG), (5, 7, ARG), (2, -1, ARG)):
        args = list(back)
        args[at] = bad
        assert L.omnihd_token_embed_bwd(*args) == status, (at, bad)
    fwd = [p, 8, 0, p, 8, 0, p, 0, p, 0, 1, 8, 5, p, 0, 1.0, 1e-6, 5, 8, p, p, p, None]
    for at, bad in ((17, -1), (18, 0), (18, 16385), (2, 1), (5, 3), (7, 4), (9, -1), (14, 9), (10, 4), (10, 0), (8, None), (12, 0), (3, None), (0, None), (19, None), (20, None)):
        args = list(fwd)
        args[at] = bad
        assert L.omnihd_block_join_fwd(*args) == ARG, (at, bad)
    need = L.omnihd_block_join_bwd_workspace_bytes(5, 8, 1, 5, 1)
    back = [p, 8, 0, p, 8, 0, p, 0, p, 0, 1, 8, 5, p, 0, 1.0, 5, 8, p, p, 8, p, 8, p, p, p, p, p, p, need, None]
    for at, bad, status in ((29, need - 1, WORKSPACE), (28, None, ARG), (18, None, ARG), (0, None, ARG), (6, None, ARG), (13, None, ARG), (3, None, ARG), (17, 20000, ARG)):
        args = list(back)
        args[at] = bad
        assert L.omnihd_block_join_bwd(*args) == status, (at, bad)
    need = L.omnihd_topk_distill_workspace_bytes(5, 8, 3, 0)
    call = [p, 0, 8, p, 0, 3, p, 1, 3, None, 5, 8, 3, 1.0, 1.0, None, None, 0, 0, p, 8, None, p, p, need, None]
    for at, bad, status in ((24, need - 1, WORKSPACE), (23, None, ARG), (10, -1, ARG), (11, 0, ARG), (11, (1 << 30) + 1, ARG), (12, 0, ARG), (12, 257, ARG), (13, 0.0, ARG), (13, float("nan"), ARG), (1, 3, ARG), (4, -1, ARG),
                            (18, 1, ARG), (2, 7, ARG), (5, 2, ARG), (8, 2, ARG), (20, 7, ARG), (0, None, ARG), (3, None, ARG), (6, None, ARG)):
        args = list(call)
        args[at] = bad
        assert L.omnihd_topk_distill(*args) == status, (at, bad)


def test_the_torch_face_loads_without_a_gpu_and_calls_the_loaded_library():
    from omnihd_amd._lib import lib, torch_ops
    face = torch_ops()
    assert face is torch_ops() and {"token_embedding", "block_join", "topk_distill"} <= set(dir(face))
    lib()
    with pytest.raises(RuntimeError):                      # CPU tensors get no further than the device guard or the library's own checks
        face.token_embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8), 1.0, -1, torch.float32)


def test_workspaces_cover_long_inputs():
    from omnihd_amd._lib import lib
    L = lib()
    assert L.omnihd_token_embed_bwd_workspace_bytes(0, 9, 8) > 0
    assert L.omnihd_token_embed_bwd_workspace_bytes((1 << 31) - 1, 32000, 64) > 2 * 4 * ((1 << 31) - 1)
    assert L.omnihd_topk_distill_workspace_bytes(0, 8, 1, 0) > 0 and L.omnihd_topk_distill_workspace_bytes(5, 8, 300, 0) == 0
    assert L.omnihd_block_join_bwd_workspace_bytes(0, 8, 0, 1, 1) > 0
