"""Edges of the operators on logits and gradients: factors below the smallest normal number, what autograd would have to follow, buffers written in place, handles that
are collected while something is captured, errors of other calls.  Against policy_oracle.py's float64, tolerances derived there."""
import gc
import threading

import numpy as np
import pytest
import torch  # noqa: F401  (before the library is first used: they share one HIP runtime)

import policy_oracle as po
from gpu_common import need_gpu, pkg

pytestmark = pytest.mark.gpu


def ops_():
    need_gpu()
    from alphazero_connect6_amd import policy_ops
    return policy_ops


def host(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("value,max_norm,kind", [(3e38, 1.0, "f32"), (3e38, 1e-7, "f32"), (1e30, 1e-12, "f32"), (1e38, 1e-30, "bf16"), (6e4, 1e-36, "f16"), (1e10, 1e-38, "f32")])
def test_clip_factor_below_the_smallest_normal(value, max_norm, kind):
    """the factor has lost bits in 32 bits, or is 0 there, and the clipped gradient is neither: the product is taken in 64 bits and rounded to f32 and to the type"""
    ops = ops_()
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]
    g = torch.full((20001,), value, device="cuda").to(dt)
    g[5] = -value / 3
    g[9] = 0
    v = host(g)
    norm = np.sqrt((v * v).sum())
    want = v * (np.float32(max_norm) / (norm + 1e-6))
    out = torch.empty_like(g)
    ops.GradClip([g], [out]).clip(max_norm)
    po.near(host(out), want, po.E32 * np.abs(want) + 2.0 ** -149, kind, "clipped")      # (f32 first: half a step, below the normal numbers of the smallest one)
    inside = ops.GradClip([g])
    inside.clip(max_norm)
    assert torch.equal(g, out)


def differentiable_calls(ops, x, t, w, b, p, d):
    lse = total = torch.zeros(4, device="cuda")
    ids = torch.zeros(4, 3, dtype=torch.int32, device="cuda")
    return {"logits": lambda v: ops.logits_process(v), "loss logits": lambda v: ops.policy_loss(v, t), "bias": lambda v: ops.logits_process(x, bias=v), "penalties": lambda v: ops.logits_process(x, history=ids, penalties=v),
            "weights": lambda v: ops.policy_loss(x, v, grad_scale=1.0), "grad weights": lambda v: ops.policy_loss_grad(x, v, lse, total, d), "dloss": lambda v: ops.policy_loss_grad(x, t, lse, total, v),
            "lse": lambda v: ops.policy_loss_grad(x, t, v, total, d), "total": lambda v: ops.policy_loss_grad(x, t, lse, v, d)}


def test_what_autograd_would_follow_is_refused():
    ops = ops_()
    x = torch.randn(4, 10, device="cuda")
    given = {"logits": x, "loss logits": x, "bias": torch.randn(4, 10, device="cuda"), "penalties": torch.ones(3, device="cuda"), "weights": torch.rand(4, 10, device="cuda"),
             "grad weights": torch.rand(4, 10, device="cuda"), "dloss": torch.ones(4, device="cuda"), "lse": torch.zeros(4, device="cuda"), "total": torch.ones(4, device="cuda")}
    calls = differentiable_calls(ops, x, torch.zeros(4, dtype=torch.int32, device="cuda"), None, None, None, torch.ones(4, device="cuda"))
    for name, call in calls.items():
        v = given[name]
        first = lambda r: r if isinstance(r, torch.Tensor) else r[0]  # noqa: E731
        want = first(call(v))
        leaf = v.clone().requires_grad_()
        for asks in (leaf, leaf * 1):
            with pytest.raises(pkg.C6Error, match="requires a gradient"):
                call(asks)
            with torch.no_grad():      # nothing is recorded: nothing is lost
                assert torch.equal(first(call(asks)), want), name
            assert torch.equal(first(call(asks.detach())), want), name
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(v.clone(), torch.ones_like(v))
            with pytest.raises(pkg.C6Error, match="tangent"):
                call(dual)
            assert torch.equal(first(call(v)), want), name


def test_writing_in_place_is_seen_by_autograd():
    """a tensor that autograd saved and one of the calls overwrites: the backward pass says so instead of using the new values"""
    ops = ops_()
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    lse = total = torch.zeros(3, device="cuda")
    up = torch.ones(3, device="cuda")

    def clip(t):
        ops.GradClip([t[:1], t[1:]]).clip(0.1)

    def clip_into(t):
        ops.GradClip([torch.ones_like(t)], [t]).clip(0.1)

    writes = [lambda t: ops.logits_process(t, out=t), lambda t: ops.logits_process(torch.ones_like(t), out=t), lambda t: ops.policy_loss(t, i, grad_scale=1.0, grad=t),
              lambda t: ops.policy_loss_grad(t, i, lse, total, up, out=t), clip, clip_into]
    for k, write in enumerate(writes):
        w = torch.ones(3, 7, device="cuda", requires_grad=True)
        saved = torch.randn(3, 7, device="cuda")
        y = (w * saved).sum()
        version = saved._version
        write(saved)
        assert saved._version > version, k
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    c, n = ops.GradClip([saved]), torch.zeros(1, device="cuda")
    before = n._version, saved._version
    c.norm(n)
    assert n._version > before[0] and saved._version == before[1]      # (only read)
    x = torch.randn(3, 7, device="cuda")
    ops.logits_process(x), ops.policy_loss(x, i, grad_scale=1.0), ops.policy_loss_grad(x, i, lse, total, up)
    assert x._version == 0


def test_clip_handles_beside_a_capture():
    """one thread captures; another makes, uses and drops handles, and the collector takes some: the capture stays whole, and so does what it captured"""
    ops = ops_()
    x = torch.randn(5000, device="cuda")
    y = torch.randn(300, device="cuda")
    made, ready, done = [], threading.Event(), threading.Event()
    errors = []

    def other():
        try:
            torch.cuda.set_device(0)
            ready.wait(60)
            for k in range(3):
                c = ops.GradClip([y])
                made.append(c.h is not None)
                if k == 1:
                    c.close()
                del c
            gc.collect()
        except BaseException as e:      # noqa: BLE001
            errors.append(e)
        finally:
            done.set()

    thread = threading.Thread(target=other)
    thread.start()
    kept, dropped = ops.GradClip([x]), ops.GradClip([y])
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    out = torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        kept.norm(out)
        with pytest.raises(pkg.C6Error, match="capture"):
            kept.close()
        with pytest.raises(pkg.C6Error, match="capture"):
            ops.GradClip([y])
        del dropped
        gc.collect()
        ready.set()
        assert done.wait(60)
    thread.join(60)
    assert not errors, errors
    assert made == [True] * 3
    for _ in range(3):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(out) - float(x.double().norm())) <= 1e-6 * float(out)
    ops.GradClip([y]).close()
    assert not ops.GradClip._late


def test_collected_clips_do_not_wait_for_the_device():
    ops = ops_()
    x = torch.randn(1000, device="cuda")
    c = ops.GradClip([x])
    n = c.norm()
    h = c.h
    del c
    gc.collect()
    assert h in ops.GradClip._late
    assert abs(float(n) - float(x.double().norm())) <= 1e-6 * float(n)
    d = ops.GradClip([x])
    assert not ops.GradClip._late and torch.equal(d.norm(), n)


def test_errors_of_other_calls_are_not_taken_for_ones_own():
    """an error that an earlier HIP call of the thread left behind: the operators' launches work and say so"""
    ops = ops_()
    x = torch.randn(5, 99, device="cuda")
    i = torch.zeros(5, dtype=torch.int32, device="cuda")
    long = torch.randn(2, 200003, device="cuda")      # (two launches)
    clip = ops.GradClip([x.clone()])
    want = [ops.logits_process(x), *ops.policy_loss(x, i, grad_scale=1.0), *ops.policy_loss(long, i[:2], grad_scale=1.0), clip.norm()]
    lse, total = want[2], want[3]
    want.append(ops.policy_loss_grad(x, i, lse, total, want[1]))
    torch.cuda.synchronize()
    hip = pkg.lib()
    calls = [lambda: [ops.logits_process(x)], lambda: list(ops.policy_loss(x, i, grad_scale=1.0)), lambda: list(ops.policy_loss(long, i[:2], grad_scale=1.0)), lambda: [clip.norm()],
             lambda: [ops.policy_loss_grad(x, i, lse, total, want[1])]]
    got = []
    try:
        for call in calls:
            assert hip.hipSetDevice(12345) != 0
            got += call()
    finally:
        hip.hipGetLastError()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("width", [7, 361, 5001, 40001, 70001])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_weights_at_illegal_entries_count_for_nothing(width, kind):
    """... whatever stands there: NaN, infinities; in every way a loss against weights goes, and in the backward pass alone"""
    ops = ops_()
    rng = np.random.default_rng(width)
    rows = 5000 if width == 7 else 6
    x = torch.tensor(rng.normal(0, 3, (rows, width)), device="cuda").to({"f32": torch.float32, "bf16": torch.bfloat16}[kind])
    keep = rng.random((rows, width)) < 0.5
    keep[1] = False
    keep[2] = False
    keep[2, width - 1] = True
    t = (rng.random((rows, width)) * keep).astype(np.float32)
    junk = np.where(keep, t, rng.choice(np.array([np.nan, np.inf, -np.inf, 3e38], np.float32), (rows, width))).astype(np.float32)
    m, clean, dirty = torch.tensor(po.pack(keep), device="cuda"), torch.tensor(t, device="cuda"), torch.tensor(junk, device="cuda")
    a, b = ops.policy_loss(x, clean, mask=m, grad_scale=0.5), ops.policy_loss(x, dirty, mask=m, grad_scale=0.5)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and all(bool(v[0 if k == 1 else slice(None)].isfinite().all()) for k, v in enumerate(a))
    assert all(torch.equal(p, q) for p, q in zip(ops.policy_loss(x, clean, mask=m), ops.policy_loss(x, dirty, mask=m)))
    up = torch.full((1,), 0.5, device="cuda")
    assert torch.equal(ops.policy_loss_grad(x, clean, a[1], a[2], up, mask=m), ops.policy_loss_grad(x, dirty, a[1], a[2], up, mask=m))
    want, tol = po.loss(host(x)[:6], t[:6], po.pack(keep)[:6], 0.5)
    po.near(host(a[3])[:6], want["grad"], tol["grad"], kind, "grad")


def test_outputs_that_overlap_an_argument_are_refused():
    ops = ops_()
    x, w = torch.randn(4, 10, device="cuda"), torch.rand(4, 10, device="cuda")
    lse, total, up = torch.zeros(4, device="cuda"), torch.ones(4, device="cuda"), torch.ones(4, device="cuda")
    wide = torch.randn(4, 30, device="cuda")
    for call in (lambda: ops.policy_loss(x, w, grad_scale=1.0, grad=w), lambda: ops.policy_loss_grad(x, w, lse, total, up, out=w), lambda: ops.logits_process(x, bias=w, out=w),
                 lambda: ops.logits_process(wide[:, :10], bias=wide[:, 5:15], out=wide[:, 10:20])):
        with pytest.raises(pkg.C6Error, match="overlaps"):
            call()
    want = ops.logits_process(wide[:, :10].clone(), bias=wide[:, 10:20].clone())
    assert torch.equal(ops.logits_process(wide[:, :10], bias=wide[:, 10:20], out=wide[:, 20:]), want)      # columns of one buffer
