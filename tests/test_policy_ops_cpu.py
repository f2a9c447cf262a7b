"""The operators on logits and gradients without a GPU: what the C entry points refuse (before they look for a device), that they do not
compute without one, and that the numpy oracle of the GPU tests agrees with PyTorch's float64."""
import ctypes as C

import numpy as np
import pytest

import policy_oracle as po
from c6amd_loader import load_package

pkg = load_package()
BAD, NO_GPU = pkg.ERR_BAD_ARG, pkg.ERR_NO_GPU
A = 1 << 20              # an address that is never followed: every call below ends before it would be


def logits(rows=4, width=10, type=0, device=0, x=A, x_stride=10, mask=None, mask_row=0, mask_byte=0):
    return pkg.Logits(rows, width, type, device, x, x_stride, mask, mask_row, mask_byte)


def process(l, history=None, hs=0, n=None, cap=0, pen=None, ps=0, bias=None, bs=0, out=4 * A, os=10):
    return pkg.lib().c6_logits_process(l, history, hs, n, cap, pen, ps, bias, bs, out, os, None)


def loss(l, target=2 * A, kind=0, ts=0, stats=3 * A, grad=None, gs=0, ws=None, nb=0):
    return pkg.lib().c6_policy_loss(l, target, kind, ts, stats, stats, stats, grad, gs, 1.0, ws, nb, None)


def grad_of(l, target=2 * A, kind=0, ts=0, lse=3 * A, total=3 * A, dloss=3 * A, ds=0, grad=4 * A, gs=10):
    return pkg.lib().c6_policy_loss_grad(l, target, kind, ts, lse, total, dloss, ds, grad, gs, None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(width=-1), dict(width=(1 << 30) + 1, x_stride=1 << 31), dict(type=3), dict(x=None), dict(x=A + 2), dict(type=1, x=A + 1), dict(x_stride=-1),
                                dict(mask_row=-1, mask=A), dict(mask_byte=-1, mask=A), dict(x_stride=1 << 62)])
def test_bad_logits_are_refused_by_every_entry_point(kw):
    l = logits(**kw)
    assert process(l) == BAD and loss(l) == BAD and grad_of(l) == BAD
    assert pkg.lib().c6_last_error().decode().startswith("logits")


def test_null_logits():
    assert process(None) == BAD and loss(None) == BAD and grad_of(None) == BAD


@pytest.mark.parametrize("kw", [dict(out=None), dict(out=4 * A + 2), dict(os=9), dict(os=-10), dict(os=1 << 62), dict(out=A, os=11), dict(out=A + 4), dict(out=A + 4 * 35),
                                dict(history=A), dict(history=A, cap=-1, pen=A), dict(history=A, cap=3, pen=A, hs=-3), dict(history=A, cap=3, pen=A, ps=-3),
                                dict(history=A + 1, cap=3, pen=A), dict(history=A, cap=3, pen=A + 2), dict(history=A, cap=3, pen=A, n=A + 1),
                                dict(history=A, cap=3, pen=A, hs=1 << 62), dict(history=A, cap=(1 << 30) + 1, pen=A), dict(bias=A, bs=-1), dict(bias=A + 3), dict(bias=A, bs=1 << 62)])
def test_bad_process_arguments(kw):
    assert process(logits(), **kw) == BAD


@pytest.mark.parametrize("kw", [dict(target=None), dict(kind=3), dict(kind=-1), dict(target=2 * A + 2), dict(kind=1, target=2 * A + 4), dict(kind=2, ts=-1), dict(kind=2, ts=1 << 62),
                                dict(stats=None), dict(stats=3 * A + 2), dict(grad=A, gs=11), dict(grad=A + 8, gs=10), dict(grad=4 * A, gs=9), dict(grad=4 * A + 1, gs=10)])
def test_bad_loss_arguments(kw):
    assert loss(logits(), **kw) == BAD


@pytest.mark.parametrize("kw", [dict(target=None), dict(kind=7), dict(lse=None), dict(total=None), dict(dloss=None), dict(dloss=A + 2), dict(ds=-1), dict(grad=None), dict(gs=3)])
def test_bad_loss_grad_arguments(kw):
    assert grad_of(logits(), **kw) == BAD


@pytest.mark.parametrize("kw", [dict(), dict(out=A), dict(out=4 * A, os=12)])
def test_sound_calls_get_as_far_as_the_device(kw):
    if pkg.device_count() > 0:
        pytest.skip("a GPU is present: the addresses are not real")
    assert process(logits(), **kw) == NO_GPU
    # rows of x and of the output interleaved in one buffer
    assert process(logits(x_stride=32), out=A + 4 * 16, os=32) == NO_GPU and process(logits(x_stride=32), out=A - 4 * 16, os=32) == NO_GPU
    assert process(logits(x_stride=32), out=A + 4 * 9, os=32) == BAD and process(logits(x_stride=32), out=A + 4 * 23, os=32) == BAD
    assert loss(logits(), grad=A, gs=10) == NO_GPU and grad_of(logits(), grad=A) == NO_GPU
    assert loss(logits(rows=0, x=None)) == NO_GPU and process(logits(width=0, x=None), out=None) == NO_GPU


def clip_create(spec, outs=True, device=0):
    """spec: (src, dst, size, type) per tensor"""
    k = len(spec)
    h = C.c_void_p()
    rc = pkg.lib().c6_clip_create(k, (C.c_void_p * k)(*[s[0] for s in spec]), (C.c_void_p * k)(*[s[1] for s in spec]) if outs else None,
                                  (C.c_size_t * k)(*[s[2] for s in spec]), (C.c_int * k)(*[s[3] for s in spec]), device, C.byref(h))
    assert rc != pkg.OK and not h.value
    return rc


def test_clip_refusals():
    L = pkg.lib()
    assert L.c6_clip_create(1, None, None, None, None, 0, C.byref(C.c_void_p())) == BAD
    assert L.c6_clip_create(-1, None, None, None, None, 0, C.byref(C.c_void_p())) == BAD
    assert L.c6_clip_create(0, None, None, None, None, 0, None) == BAD
    assert L.c6_clip_norm(None, A, A, 8, None) == BAD and L.c6_clip_apply(None, 1.0, A, A, 8, None) == BAD
    assert L.c6_clip_workspace(None) == 0
    L.c6_clip_destroy(None)
    for spec in ([(A, A, 4, 3)], [(None, A, 4, 0)], [(A, None, 4, 0)], [(A + 2, A + 2, 4, 0)], [(A, A + 1, 4, 1)], [(A, A, 1 << 60, 0)],
                 [(A, A, 4, 0), (A, A, 4, 0)],                       # the same tensor twice: it would be scaled twice
                 [(A, A, 4, 0), (A + 8, A + 8, 4, 0)],               # ... in part
                 [(A, A + 8, 4, 0)], [(A, 2 * A, 4, 0), (3 * A, 2 * A + 12, 4, 0)], [(A, 2 * A, 100, 0), (2 * A, 3 * A, 1, 0)]):
        assert clip_create(spec) == BAD, spec
    assert clip_create([(A, None, 4, 0), (A + 12, None, 2, 0)], outs=False) == BAD


def test_clip_sound_tables_get_as_far_as_the_device():
    if pkg.device_count() > 0:
        pytest.skip("a GPU is present: the addresses are not real")
    for spec in ([(A, A, 4, 0), (A + 16, A + 16, 3, 1)], [(A, 2 * A, 4, 0), (A, 3 * A, 4, 0)], [(None, None, 0, 2)], [(A, A, 4, 2), (A, A, 0, 0)]):
        assert clip_create(spec) == NO_GPU, spec


def test_trainer_refusals_without_a_trainer():
    L = pkg.lib()
    f = C.c_float()
    assert L.c6_trainer_set_policy_loss(None, 0) == BAD and L.c6_trainer_set_clip(None, 1.0) == BAD and L.c6_trainer_grad_norm(None, C.byref(f)) == BAD
    assert L.c6_replay_sample_device_pi(None, 1, 0, 0, None, None, None, None, None, None) == BAD


def test_python_face_refuses_host_tensors():
    import torch
    from alphazero_connect6_amd import policy_ops as ops
    x = torch.zeros(2, 5)
    for call in (lambda: ops.logits_process(x), lambda: ops.policy_loss(x, torch.zeros(2, dtype=torch.int32)), lambda: ops.GradClip([x]), lambda: ops.GradClip([])):
        with pytest.raises(pkg.C6Error):
            call()


def test_oracle_against_torch():
    import torch
    rng = np.random.default_rng(0)
    x = rng.normal(0, 3, (6, 37))
    keep = rng.random((6, 37)) < 0.5
    keep[2] = False
    keep[3] = False
    keep[3, 36] = True
    t = rng.random((6, 37))
    out, _ = po.loss(x, t, po.pack(keep), scale=0.25)
    xt = torch.tensor(x, requires_grad=True)
    masked = xt.masked_fill(~torch.tensor(keep), -np.inf)
    w = torch.tensor(t) * torch.tensor(keep)
    lp = torch.log_softmax(masked, 1)
    ref = -(w * lp.masked_fill(~torch.tensor(keep), 0.0)).sum(1)
    live = [r for r in range(6) if r != 2]
    (g,) = torch.autograd.grad(0.25 * ref[live].sum(), xt)
    g = g.detach().numpy()
    g[2] = 0
    assert np.abs(out["loss"][live] - ref[live].detach().numpy()).max() < 1e-12 and out["loss"][2] == 0 and out["lse"][2] == -np.inf
    assert np.abs(out["grad"] - g).max() < 1e-14
    h, _ = po.grad_from(x, t, out["lse"], out["total"], 0.25, po.pack(keep))
    assert np.abs(h - g).max() < 1e-14
    # the gradient by differences
    for r, v in ((0, int(np.argmax(keep[0]))), (3, 36), (5, int(np.argmax(keep[5])))):
        e = np.zeros_like(x)
        e[r, v] = 1e-5
        d = (po.loss(x + e, t, po.pack(keep))[0]["loss"] - po.loss(x - e, t, po.pack(keep))[0]["loss"])[r] / 2e-5
        assert abs(0.25 * d - out["grad"][r, v]) < 1e-8


def test_a_trainers_error_is_not_hidden_behind_an_older_one():
    L = pkg.lib()
    assert process(None) == BAD and b"logits" in L.c6_last_error()
    assert L.c6_trainer_set_clip(None, 1.0) == BAD
    assert b"c6_trainer_set_clip" in L.c6_last_error() and b"c6_trainer_set_clip" in L.c6_trainer_last_error()
