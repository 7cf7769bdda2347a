"""CPU: the refusals of the gradient norm, the clipping and the clipped step -- at the Python surface and at the C ABI -- and what
they do without gradients."""
import ctypes as C
import math

import pytest
import torch

from vegs_amd import _capi, optim


def _with_grad(g):
    p = torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype))
    p.grad = g
    return p


def test_cpu_gradients_are_refused():
    p = _with_grad(torch.ones(5))
    with pytest.raises(ValueError, match="GPU"):
        optim.grad_norm([p])
    with pytest.raises(ValueError, match="GPU"):
        optim.clip_grad_norm_([p], 1.0)
    opt = optim.Adam([p], lr=1e-3)
    with pytest.raises(ValueError, match="GPU"):
        optim.step_many([opt], max_grad_norm=1.0)
    assert not opt.state and torch.equal(p.grad, torch.ones(5))


def test_no_gradients_give_a_zero():
    p = torch.nn.Parameter(torch.zeros(3))
    assert optim.grad_norm([p]).item() == 0.0
    assert optim.clip_grad_norm_(p, 1.0).item() == 0.0
    assert optim.clip_grad_norm_([], 1.0).item() == 0.0


@pytest.mark.parametrize("max_norm", [-1.0, math.nan])
def test_bad_bounds_are_refused(max_norm):
    p = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grad_norm_([p], max_norm)
    with pytest.raises(ValueError, match="max_norm"):
        optim.step_many([optim.Adam([p])], max_grad_norm=max_norm)


def test_other_norms_are_refused():
    p = torch.nn.Parameter(torch.zeros(3))
    for norm_type in (1.0, 0.5, 3):
        with pytest.raises(NotImplementedError):
            optim.grad_norm([p], norm_type)
    with pytest.raises(ValueError):
        optim.step_many([optim.Adam([p])], grad_norm=torch.tensor(1.0))


def test_c_entries_refuse_bad_tables():
    lib = _capi.load()
    some = 1 << 20                                        # (a made-up address: nothing is launched for a refused call)

    def table(*entries):
        flat = [x for e in entries for x in e]
        return (C.c_int64 * max(len(flat), 1))(*flat), len(entries)

    for entries in ([(0, 4, 0)], [(some, -1, 0)], [(some, 4, 3)], [(some, 4, -1)], [(some + 2, 4, 0)], [(some + 1, 4, 1)],
                    [(some, 1 << 41, 0)], [(some, 4, 0), (0, 1, 2)]):
        t, n = table(*entries)
        assert lib.vr_grad_norm(t, n, None, 0, 2, some, some, None) == -1, entries
        assert lib.vr_clip_grads(t, n, some, 1.0, None) == -1, entries
        assert lib.vr_clip_grad_norm(t, n, 2, 1.0, some, some, None) == -1, entries
        assert b"tensor" in lib.vr_last_error()
    t, n = table((some, 4, 0))
    assert lib.vr_grad_norm(t, n, None, 0, 1, some, some, None) == -1           # the norm types are 2 and 0
    assert lib.vr_grad_norm(t, n, None, 0, 2, None, some, None) == -1
    assert lib.vr_grad_norm(t, n, None, 0, 2, some, some + 4, None) == -1       # scratch alignment
    assert lib.vr_grad_norm(t, n, None, 1, 2, some, some, None) == -1
    assert lib.vr_grad_norm(t, -1, None, 0, 2, some, some, None) == -1
    bad = _capi.VrShGradFactors(some, some, some, 0, 5, 1, 4, 1.0)              # SH degree 4
    assert lib.vr_grad_norm(t, n, C.byref(bad), 1, 2, some, some, None) == -1
    for bound in (-1.0, math.nan):
        assert lib.vr_clip_grads(t, n, some, bound, None) == -1
        assert lib.vr_clip_grad_norm(t, n, 2, bound, some, some, None) == -1
        assert lib.vr_adam_step_clipped(None, 0, 0.9, 0.999, 1e-8, some, bound, None) == -1
    assert lib.vr_clip_grads(t, n, None, 1.0, None) == -1
    assert lib.vr_adam_step_clipped(None, 0, 0.9, 0.999, 1e-8, None, 1.0, None) == -1
    assert lib.vr_sh_adam_step_clipped(None, 0, None, None, 1, 0, 0, 1, 1.0, None, None, 0.9, 0.999, 1e-8, None, 1.0, None) == -1


def test_scratch_grows_with_the_launches():
    lib = _capi.load()
    one = lib.vr_grad_norm_scratch_bytes(0, 0)
    assert one > 0 and one % 8 == 0
    assert lib.vr_grad_norm_scratch_bytes(128, 0) == one and lib.vr_grad_norm_scratch_bytes(129, 0) == 2 * one
    assert lib.vr_grad_norm_scratch_bytes(1, 3) == 4 * one


def test_gradients_that_fill_their_memory_are_told_from_others():
    t = torch.zeros(4, 6, 5)
    assert optim._dense(t) and optim._dense(t.permute(2, 0, 1)) and optim._dense(t[1]) and optim._dense(t[:, :1].squeeze(1)[:0])
    assert not optim._dense(t[:, ::2]) and not optim._dense(t[:, :, 1:]) and not optim._dense(torch.zeros(1).expand(7))
    assert optim._dense(t[:, :1, :1][:1])                # one element: its strides say nothing


def test_sparse_gradients_are_refused():
    p = torch.nn.Parameter(torch.zeros(4, 3))
    p.grad = torch.sparse_coo_tensor([[1]], [[1.0, 2.0, 3.0]], (4, 3))
    with pytest.raises(ValueError, match="dense"):
        optim.grad_norm([p])
    with pytest.raises(ValueError, match="dense"):
        optim.clip_grad_norm_([p], 1.0)


def test_gradients_are_told_apart_by_their_elements():
    b = torch.zeros(12)
    assert len(optim._once([b[:4], b[::2][:4]])) == 2             # one address and one number of elements, other elements
    assert len(optim._once([b[:4], b[:4], b[:4].reshape(2, 2), b[:4].reshape(2, 2).t()])) == 1
    assert len(optim._once([b[::2], b[::2], b[::3][:4], b[::2][:4]])) == 3
    assert len(optim._once([b[:4], b.view(torch.int32)[:4]])) == 2


def test_c_entries_refuse_to_scale_shared_memory():
    """(Made-up addresses: nothing is launched for a refused call.)"""
    lib = _capi.load()
    some = 1 << 20

    def table(*entries):
        return (C.c_int64 * (3 * len(entries)))(*[x for e in entries for x in e]), len(entries)

    many = [(some + 4096 * i, 1024, 0) for i in range(300)]
    for entries in ([(some, 8, 0), (some, 8, 0)], [(some, 8, 0), (some + 28, 1, 0)], [(some + 28, 5, 0), (some, 8, 0)],
                    [(some, 9, 1), (some + 16, 4, 0)], [(some, 100, 0), (some + 1000, 5, 0), (0, 0, 0), (some + 200, 3, 1)],
                    many + [(some + 4096 * 200 + 4092, 1, 0)]):
        t, n = table(*entries)
        for rc in (lib.vr_clip_grads(t, n, some, 1.0, None), lib.vr_clip_grad_norm(t, n, 2, 1.0, some, some, None)):
            assert rc == -1 and b"share memory" in lib.vr_last_error()


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("bound", [-1.0, math.nan])
def test_the_trainer_refuses_a_bad_bound_before_anything_else(bound, fused):
    from vegs_amd import iteration
    with pytest.raises(ValueError, match="max_norm"):
        iteration.Trainer(None, torch.device("cpu"), fused=fused, max_grad_norm=bound)
