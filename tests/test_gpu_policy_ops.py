"""The operators on logits and gradients (csrc/policy_ops.hip, grad_clip.hip) against policy_oracle.py's float64, through the Python face on
device tensors.  Tolerances: policy_oracle.py derives them, the last rounding of the type included."""
import numpy as np
import pytest
import torch  # noqa: F401  (before the library is first used: they share one HIP runtime)

import policy_oracle as po
from gpu_common import need_gpu, pkg

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "bf16"]
LOWEST = {"f32": -3.4028234663852886e38, "f16": -65504.0, "bf16": -3.3895313892515355e38}


def setup():
    need_gpu()
    import torch
    from alphazero_connect6_amd import policy_ops
    return torch, policy_ops, {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def host(t):
    return t.detach().double().cpu().numpy()


def strided(torch, rows, width, dtype, pad, lead, device="cuda"):
    """an uninitialised [rows, width] view whose rows are `pad` apart beyond width and start `lead` elements into a buffer"""
    return torch.empty(lead + rows * (width + pad) + 8, dtype=dtype, device=device)[lead:lead + rows * (width + pad)].view(rows, width + pad)[:, :width]


def make(rows, width, kind, seed, mask="rows", pad=0, lead=0):
    """(x on the GPU, its values, mask on the GPU or None, its bytes or None); one row has nothing legal, one a single entry, and masked places hold
    the type's lowest value, infinities and NaN"""
    torch, _, dts = setup()
    rng = np.random.default_rng(seed)
    vals = rng.normal(0, 3, (rows, width))
    keep = rng.random((rows, width)) < rng.random((rows, 1))
    if rows > 2:
        keep[1] = False
        keep[2] = False
        keep[2, width - 1] = True
    if mask == "shared":
        keep[:] = keep[-1:]
    if mask != "none":
        junk = rng.integers(0, 40, (rows, width))
        for k, j in enumerate((LOWEST[kind], np.inf, -np.inf, np.nan)):
            vals[~keep & (junk == k)] = j
    x = strided(torch, rows, width, dts[kind], pad, lead)
    x.copy_(torch.tensor(vals, device="cuda"))
    if mask == "none":
        return x, host(x), None, None
    packed = po.pack(keep if mask != "shared" else keep[:1])
    m = torch.tensor(packed, device="cuda")
    if mask == "soa":
        m = m.t().contiguous().t()
    return x, host(x), m, packed


SHAPES = [(1, 1), (3, 2), (4, 7), (5, 8), (3, 64), (6, 81), (130, 225), (9, 361), (4, 1000), (3, 4096), (3, 8193), (2, 20001), (3, 100003)]
MASKS = ["none", "rows", "soa", "shared"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("i,shape", list(enumerate(SHAPES)), ids=lambda s: str(s))
def test_process(i, shape, kind):
    torch, ops, _ = setup()
    rows, width = shape
    rng = np.random.default_rng(100 + i)
    x, vals, m, packed = make(rows, width, kind, i, MASKS[i % 4], pad=(i * 3) % 5, lead=i % 3)
    cap = [0, 1, 5, 300, 5000][i % 5]
    hist = rng.integers(-1, width + 1, (rows, cap)).astype(np.int32)          # -1 and width: outside
    if cap > 4:
        hist[0, :5] = [np.iinfo(np.int32).max, np.iinfo(np.int32).min, 0, 0, width - 1]
    lens = rng.integers(-1, cap + 2, rows).astype(np.int32)                   # below none and beyond all
    if cap:
        lens[0] = cap
    pen = np.stack([rng.uniform(0.5, 2, rows), rng.uniform(-0.5, 0.5, rows), rng.uniform(0, 1, rows)], 1).astype(np.float32)
    bias = rng.normal(0, 2, (rows, width) if i % 2 else (width,)).astype(np.float32)
    bias.reshape(-1)[0] = -np.inf
    g = lambda a: torch.tensor(a, device="cuda")  # noqa: E731
    for case in ({}, {"bias": bias}, {"history": hist, "history_len": lens, "penalties": pen}, {"history": hist[:1], "penalties": pen[0], "bias": bias},
                 {"history": hist, "penalties": pen[:1]}):
        want, tol = po.process(vals, packed, **case)
        dev = {k: g(v) for k, v in case.items()}
        keep = x.clone()
        y = ops.logits_process(x, mask=m, **dev)
        assert y.is_contiguous() and y.dtype == x.dtype
        po.near(host(y), want, tol, kind, ("process", shape, kind, list(case)))
        assert torch.equal(keep.nan_to_num(nan=99.0), x.nan_to_num(nan=99.0))
        # into a view with other strides, nothing between its rows touched; then in place: the same bits
        buf = torch.full((rows, width + 3), 7.0, dtype=x.dtype, device="cuda")
        z = ops.logits_process(x, mask=m, out=buf[:, 1:width + 1], **dev)
        assert z.data_ptr() == buf.data_ptr() + buf.element_size()
        assert torch.equal(z.nan_to_num(nan=99.0), y.nan_to_num(nan=99.0)) and bool((buf[:, 0] == 7).all()) and bool((buf[:, width + 1:] == 7).all())
        w = strided(torch, rows, width, x.dtype, (i * 3) % 5, i % 3)
        w.copy_(x)
        assert ops.logits_process(w, mask=m, out=w, **dev) is w
        assert torch.equal(w.nan_to_num(nan=99.0), y.nan_to_num(nan=99.0))


# Many narrow rows: from 4096 rows (8192 with a history) of up to 384 entries on, 16 lanes take a row; a case on each side of each border.  The history's
# room: too small for one 16-byte load, just enough, ragged, longer than what the lanes of a row read at once.
@pytest.mark.parametrize("rows,width,kind,mask,cap", [
    (4095, 361, "f32", "rows", 3), (4096, 361, "f32", "soa", 4), (8191, 225, "bf16", "rows", 63), (8192, 225, "bf16", "soa", 64), (8193, 361, "f16", "shared", 65),
    (8192, 384, "f32", "none", 200), (8192, 385, "f32", "rows", 200), (9001, 81, "f32", "soa", 50), (8200, 3, "bf16", "rows", 7), (8192, 7, "f16", "rows", 1),
    (10001, 8, "f32", "shared", 5), (8197, 361, "bf16", "rows", 700), (8192, 1, "f32", "rows", 2), (8200, 383, "f32", "soa", 3)], ids=str)
def test_process_of_many_rows(rows, width, kind, mask, cap):
    torch, ops, _ = setup()
    rng = np.random.default_rng(rows + width + cap)
    x, vals, m, packed = make(rows, width, kind, width, mask, pad=width % 4, lead=cap % 3)
    hist = rng.integers(-1, width + 1, (rows, cap)).astype(np.int32)
    lens = rng.integers(-1, cap + 2, rows).astype(np.int32)
    pen = np.stack([rng.uniform(0.5, 2, rows), rng.uniform(-0.5, 0.5, rows), rng.uniform(0, 1, rows)], 1).astype(np.float32)
    bias = rng.normal(0, 2, (rows, width)).astype(np.float32)
    for case in ({}, {"bias": bias[0]}, {"history": hist, "history_len": lens, "penalties": pen}, {"history": hist, "penalties": pen[0], "bias": bias}):
        want, tol = po.process(vals, packed, **case)
        dev = {k: torch.tensor(v, device="cuda") for k, v in case.items()}
        y = ops.logits_process(x, mask=m, **dev)
        po.near(host(y), want, tol, kind, ("process", rows, width, kind, list(case)))
        buf = torch.full((rows, width + 3), 7.0, dtype=x.dtype, device="cuda")
        z = ops.logits_process(x, mask=m, out=buf[:, 1:width + 1], **dev)
        assert torch.equal(z.nan_to_num(nan=99.0), y.nan_to_num(nan=99.0)) and bool((buf[:, 0] == 7).all()) and bool((buf[:, width + 1:] == 7).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("target", ["index32", "index64", "weights"])
@pytest.mark.parametrize("i,shape", list(enumerate(SHAPES)), ids=lambda s: str(s))
def test_loss_and_gradient(i, shape, target, kind):
    torch, ops, _ = setup()
    rows, width = shape
    rng = np.random.default_rng(200 + i)
    x, vals, m, packed = make(rows, width, kind, 50 + i, MASKS[(i + len(target)) % 4], pad=(i * 3) % 5, lead=i % 3)
    if target == "weights":
        t = (rng.random((rows, width)) ** 4 * rng.uniform(0, 30, (rows, 1))).astype(np.float32)
        t[rng.random((rows, width)) < 0.5] = 0
        t[-1] = 0
        td = strided(torch, rows, width, torch.float32, i % 4, i % 2)
        td.copy_(torch.tensor(t, device="cuda"))
    else:
        t = rng.integers(0, width, rows).astype(np.int32 if target == "index32" else np.int64)
        if packed is not None:      # a legal entry for most, an illegal one for some
            ok = po.legal(packed, rows, width)
            for r in range(rows):
                if ok[r].any() and r % 5 != 4:
                    t[r] = rng.choice(np.flatnonzero(ok[r]))
        if rows > 4:
            t[3], t[4] = -1, width
            if target == "index64":
                t[4] = (1 << 32) + t[0]
        td = torch.tensor(t, device="cuda")
    scale = 1.0 / rows
    want, tol = po.loss(vals, t, packed, np.float32(scale))
    got = ops.policy_loss(x, td, mask=m, grad_scale=scale)
    names = ("loss", "lse", "total")
    for k, v in zip(names, got):
        po.near(host(v), want[k], tol[k], "f32", (k, shape, kind, target))
    po.near(host(got[3]), want["grad"], tol["grad"], kind, ("grad", shape, kind, target))
    fwd = ops.policy_loss(x, td, mask=m)
    assert len(fwd) == 3 and all(torch.equal(a, b) for a, b in zip(fwd, got))
    # the backward pass alone, an upstream gradient per row and one for all
    up = torch.tensor(rng.uniform(0.5, 1.5, rows), dtype=torch.float32, device="cuda")
    for d in (up, up[:1].clone()):
        g = ops.policy_loss_grad(x, td, got[1], got[2], d, mask=m)
        w, wt = po.grad_from(vals, t, host(got[1]), host(got[2]), host(d), packed)
        po.near(host(g), w, wt, kind, ("backward", shape, kind, target))
    # in place: the same bits
    loss_into = lambda z, o: ops.policy_loss(z, td, mask=m, grad_scale=scale, grad=o)[3]  # noqa: E731
    back_into = lambda z, o: ops.policy_loss_grad(z, td, got[1], got[2], up, mask=m, out=o)  # noqa: E731
    for f in (loss_into, back_into):
        z = strided(torch, rows, width, x.dtype, (i * 3) % 5, i % 3)
        z.copy_(x)
        ref = f(x, None)
        assert f(z, z) is z and torch.equal(z, ref)


# Which way a loss goes depends on rows and width (policy_ops.hip, splits() and loss_launch()): four rows a wave from 4096 rows on, 16 to 1024 lanes a row, rows that a
# workgroup takes one after the other, rows split into chunks.  (rows, width, type, target, mask): a case on each side of each border.
WAYS = [(4096, 81, "f32", "index32", "rows"), (4097, 225, "bf16", "weights", "soa"), (4099, 361, "f16", "weights", "shared"), (5000, 384, "f32", "index64", "none"),
        (4096, 385, "f32", "weights", "rows"), (4095, 361, "bf16", "weights", "rows"), (4100, 768, "bf16", "index32", "rows"), (4100, 769, "bf16", "index32", "none"),
        (70, 1024, "f32", "weights", "none"), (70, 1025, "f32", "weights", "rows"), (300, 4097, "f16", "weights", "rows"), (300, 8192, "f32", "index32", "rows"),
        (300, 8193, "f32", "weights", "rows"), (600, 16385, "f32", "index32", "none"), (520, 40001, "bf16", "weights", "shared"), (300, 65536, "bf16", "weights", "none"),
        (300, 65537, "bf16", "weights", "rows"), (300, 65537, "bf16", "index32", "rows"), (129, 65536, "f32", "index64", "rows"), (130, 65537, "f32", "index32", "none"),
        (128, 32769, "f32", "index32", "rows"), (129, 32769, "f32", "index32", "rows"), (257, 131072, "f16", "index32", "none"), (2, 1000003, "bf16", "weights", "rows"),
        (257, 99001, "bf16", "index64", "rows"), (300, 50001, "f32", "index32", "soa"), (320, 98313, "f16", "index64", "shared"), (321, 98313, "f16", "index32", "rows"),
        (256, 50001, "f32", "index32", "rows"), (513, 49157, "f32", "index32", "rows"),
        (300, 12288, "f32", "weights", "rows"), (300, 12289, "f32", "weights", "rows"), (300, 24576, "bf16", "index32", "soa"), (300, 24577, "bf16", "weights", "none"),
        (300, 24576, "f32", "index64", "rows"), (300, 24577, "f32", "weights", "rows"), (300, 49153, "f16", "index32", "none"), (300, 49152, "bf16", "weights", "rows"),
        (300, 49152, "f32", "index32", "rows"), (300, 98305, "bf16", "index64", "none"), (300, 57344, "f32", "index64", "none"), (300, 114689, "f16", "index32", "rows"),
        (2, 9000001, "f32", "index32", "rows"), (1, 9000001, "f16", "weights", "none")]      # (more chunks than workgroups a row)


@pytest.mark.parametrize("rows,width,kind,target,mask", WAYS)
def test_every_way_a_loss_goes(rows, width, kind, target, mask):
    torch, ops, _ = setup()
    rng = np.random.default_rng(rows + width)
    x, vals, m, packed = make(rows, width, kind, rows * 7 + width, mask)
    if target == "weights":
        t = (rng.random((rows, width)) ** 6).astype(np.float32)
        t[5:9] = 0
    else:
        t = rng.integers(0, width, rows).astype(np.int32 if target == "index32" else np.int64)
    td = torch.tensor(t, device="cuda")
    before = x.clone()
    got = ops.policy_loss(x, td, mask=m, grad_scale=0.5)
    fwd = ops.policy_loss(x, td, mask=m)
    assert torch.equal(x.nan_to_num(nan=99.0), before.nan_to_num(nan=99.0))
    pick = np.unique(np.r_[:min(rows, 12), rng.integers(0, rows, 40), rows - 1])      # these rows against float64, all of them against one another
    sub = packed if packed is None or packed.shape[0] == 1 else packed[pick]
    want, tol = po.loss(vals[pick], t[pick], sub, 0.5)
    idx = torch.tensor(pick, device="cuda")
    for k, v in zip(("loss", "lse", "total"), got):
        po.near(host(v[idx]), want[k], tol[k], "f32", k)
    po.near(host(got[3][idx]), want["grad"], tol["grad"], kind, "grad")
    # the forward pass alone may go another way: as far apart as two roundings
    for k, a, b in zip(("loss", "lse", "total"), fwd, got):
        po.near(host(a[idx]), want[k], tol[k], "f32", k + " alone")
        fin = torch.isfinite(b)
        assert torch.equal(torch.isfinite(a), fin) and bool(((a - b)[fin].abs() <= 1e-4 * (1 + b[fin].abs())).all())
    # the backward pass alone agrees over ALL rows
    g = ops.policy_loss_grad(x, td, got[1], got[2], torch.full((1,), 0.5, device="cuda"), mask=m)
    d = (g.float() - got[3].float()).abs()
    assert bool((d <= 2 * po.HALF_STEP[kind] * (g.float().abs() + got[3].float().abs()) + 2e-5 * got[2][:, None] + po.TINY[kind]).all())
    # in place
    z = x.clone()
    assert torch.equal(ops.policy_loss(z, td, mask=m, grad_scale=0.5, grad=z)[3], got[3])


@pytest.mark.parametrize("width", [5, 300, 40000])
def test_rows_with_infinities_and_nan(width):
    """what stands at LEGAL entries: -infinity is an entry of probability 0, +infinity and NaN make the row NaN, a row of nothing but -infinity is empty"""
    torch, ops, _ = setup()
    x = torch.zeros(7, width, device="cuda")
    x[0] = -np.inf
    x[1, 1:] = -np.inf
    x[2, 2] = np.inf
    x[3, 3] = np.nan
    x[4] = np.nan
    x[5] = LOWEST["f32"]
    x[6] = 3e38
    t = torch.zeros(7, dtype=torch.int32, device="cuda")
    loss, lse, total, grad = [host(v) for v in ops.policy_loss(x, t, grad_scale=1.0)]
    assert loss[0] == 0 and lse[0] == -np.inf and total[0] == 0 and (grad[0] == 0).all()
    assert loss[1] == 0 and lse[1] == 0 and total[1] == 1 and (grad[1] == 0).all()
    for r in (2, 3, 4):
        assert np.isnan(loss[r]) and np.isnan(lse[r]) and np.isnan(grad[r]).any()
    for r in (5, 6):      # log(width) is lost beside 3e38, in the sum but not in the loss
        assert abs(loss[r] - np.log(width)) < 1e-5 * np.log(width) and np.isfinite(lse[r]) and abs(grad[r, 1] - 1 / width) < 1e-5 / width
    t[1] = 1              # the move played has probability 0: the loss is infinite, the gradient is not
    loss, _, total, grad = [host(v) for v in ops.policy_loss(x, t, grad_scale=1.0)]
    assert loss[1] == np.inf and total[1] == 1 and grad[1, 1] == -1 and grad[1, 0] == 1
    w = torch.zeros(7, width, device="cuda")
    w[:, 0] = 2.0
    w[1, 4] = 3.0
    loss, _, total, grad = [host(v) for v in ops.policy_loss(x, w, grad_scale=1.0)]
    assert loss[1] == np.inf and total[1] == 5 and loss[0] == 0 and total[0] == 0 and grad[1, 4] == -3 and grad[1, 0] == 3


def test_nothing_to_do():
    torch, ops, _ = setup()
    e = torch.empty(0, 9, device="cuda")
    assert ops.logits_process(e).shape == (0, 9)
    assert [v.shape[0] for v in ops.policy_loss(e, torch.empty(0, dtype=torch.int64, device="cuda"), grad_scale=1.0)] == [0, 0, 0, 0]
    w = torch.empty(3, 0, device="cuda")
    assert ops.logits_process(w).shape == (3, 0)
    loss, lse, total, grad = ops.policy_loss(w, torch.zeros(3, dtype=torch.int32, device="cuda"), grad_scale=1.0)
    assert host(loss).tolist() == [0] * 3 and host(lse).tolist() == [-np.inf] * 3 and host(total).tolist() == [0] * 3 and grad.shape == (3, 0)
    assert ops.policy_loss_grad(w, torch.zeros(3, 0, device="cuda"), lse, total, loss).shape == (3, 0)


def test_broadcast_logits_and_rows_behind_the_last():
    torch, ops, _ = setup()
    row = torch.randn(1, 777, device="cuda")
    t = torch.arange(9, dtype=torch.int32, device="cuda")
    a = ops.policy_loss(row.expand(9, 777), t, grad_scale=0.5)
    b = ops.policy_loss(row.repeat(9, 1), t, grad_scale=0.5)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert torch.equal(ops.logits_process(row.expand(9, 777)), row.repeat(9, 1))
    buf = torch.full((12, 777), 5.0, device="cuda")
    ops.policy_loss(row.expand(9, 777), t, grad_scale=0.5, grad=buf[:9])
    assert torch.equal(buf[:9], b[3]) and bool((buf[9:] == 5).all())


def test_offsets_beyond_32_bits():
    torch, ops, _ = setup()
    far = (1 << 31) + 12345                        # elements from row to row: the second row begins beyond 2^32 bytes, the third beyond 2^32 elements
    big = torch.empty(2 * far + 1000, dtype=torch.bfloat16, device="cuda")
    x = big.as_strided((3, 1000), (far, 1))
    x.copy_(torch.randn(3, 1000, device="cuda"))
    t = torch.tensor([3, 5, 7], dtype=torch.int32, device="cuda")
    a, b = ops.policy_loss(x, t, grad_scale=1.0), ops.policy_loss(x.contiguous(), t, grad_scale=1.0)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert torch.equal(ops.logits_process(x), x.contiguous())
    ops.logits_process(a[3], out=x)
    assert torch.equal(x, a[3])
    del big, x


def test_legal_mask_of_the_board_kernel_goes_straight_in():
    """c6_legal_mask's packed layout (byte-major, game index minor) as the mask of a batch of positions, some of them full"""
    torch, ops, _ = setup()
    rng = np.random.default_rng(3)
    n, games = 15, 37
    boards = rng.integers(-1, 2, (games, n * n)).astype(np.int8)
    boards[5] = 1
    mask = pkg.legal_mask(n, pkg.to_soa(boards))
    x = rng.normal(0, 2, (games, n * n)).astype(np.float32)
    y = host(ops.logits_process(torch.tensor(x, device="cuda"), mask=torch.tensor(mask, device="cuda").t()))
    assert np.array_equal(y, np.where(boards == 0, x.astype(np.float64), -np.inf))


def test_masks_and_histories_of_any_stride():
    """rows of masks, histories, penalties and biases out of larger buffers; bits behind the row's end mean nothing"""
    torch, ops, _ = setup()
    rng = np.random.default_rng(11)
    for rows, width in ((6, 85), (5, 5003)):
        x = rng.normal(0, 2, (rows, width)).astype(np.float32)
        keep = rng.random((rows, width)) < 0.5
        packed = po.pack(keep)
        noisy = packed.copy()
        noisy[:, -1] |= (0xff << (width % 8)) & 0xff
        hist = rng.integers(0, width, (rows, 33)).astype(np.int32)
        pen = rng.uniform(0.5, 1.5, (rows, 3)).astype(np.float32)
        bias = rng.normal(0, 1, (rows, width)).astype(np.float32)

        def inside(a):      # a in the middle of a buffer twice as large
            buf = torch.zeros((a.shape[0] * 2, a.shape[1] + 7), dtype=torch.tensor(a).dtype, device="cuda")
            v = buf[::2, 3:3 + a.shape[1]]
            v.copy_(torch.tensor(a))
            return v
        wide = torch.zeros((rows, packed.shape[1] * 3), dtype=torch.uint8, device="cuda")
        wide[:, ::3] = torch.tensor(noisy, device="cuda")
        want, tol = po.process(x, packed, bias=bias, history=hist, penalties=pen)
        xd = torch.tensor(x, device="cuda")
        for m in (inside(noisy), wide[:, ::3], torch.tensor(noisy, device="cuda")):
            y = ops.logits_process(xd, mask=m, bias=inside(bias), history=inside(hist), penalties=inside(pen))
            po.near(host(y), want, tol, "f32", "strides")
            t = torch.zeros(rows, dtype=torch.int64, device="cuda")
            lw, lt = po.loss(x, t.cpu().numpy(), packed, 1.0)
            got = ops.policy_loss(inside(x), t, mask=m, grad_scale=1.0)
            po.near(host(got[0]), lw["loss"], lt["loss"], "f32", "loss")
            po.near(host(got[3]), lw["grad"], lt["grad"], "f32", "grad")


def test_two_at_once():
    """the same logits on two streams, rows split into chunks on both: a workspace each"""
    torch, ops, _ = setup()
    x = torch.randn(4, 200003, device="cuda")
    t = torch.tensor([0, 7, 200002, 9], dtype=torch.int32, device="cuda")
    want = ops.policy_loss(x, t, grad_scale=1.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.policy_loss(x, t, grad_scale=1.0))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_python_refusals():
    torch, ops, _ = setup()
    x = torch.zeros(4, 10, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    m = torch.zeros(4, 2, dtype=torch.uint8, device="cuda")
    f = torch.zeros(4, device="cuda")
    bad = [lambda: ops.logits_process(x.double()), lambda: ops.logits_process(x[0]), lambda: ops.logits_process(x.t()), lambda: ops.logits_process(x.clone().requires_grad_()),
           lambda: ops.logits_process(x, mask=m.cpu()), lambda: ops.logits_process(x, mask=m[:, :1]), lambda: ops.logits_process(x, mask=m[:3]), lambda: ops.logits_process(x, mask=m.int()),
           lambda: ops.logits_process(x, bias=f), lambda: ops.logits_process(x, bias=x.half()), lambda: ops.logits_process(x, history=m.int()),
           lambda: ops.logits_process(x, penalties=f[:3]), lambda: ops.logits_process(x, history=m, penalties=f[:3]), lambda: ops.logits_process(x, history=m.int(), penalties=f),
           lambda: ops.logits_process(x, history=m.int(), penalties=f[:3], history_len=i[:2]), lambda: ops.logits_process(x, out=x.half()), lambda: ops.logits_process(x, out=x[:2]),
           lambda: ops.logits_process(x[:, :8], out=x[:, 2:]), lambda: ops.logits_process(x, out=x[:1].expand(4, 10)),
           lambda: ops.policy_loss(x, i[:3]), lambda: ops.policy_loss(x, f), lambda: ops.policy_loss(x, x.half()), lambda: ops.policy_loss(x, x[:, :9]), lambda: ops.policy_loss(x, i, grad=x),
           lambda: ops.policy_loss(x, i.cpu()), lambda: ops.policy_loss_grad(x, i, f[:2], f, f), lambda: ops.policy_loss_grad(x, i, f, f, f[:2]), lambda: ops.policy_loss_grad(x, i, f.double(), f, f),
           lambda: ops.GradClip([x.t()]), lambda: ops.GradClip([x, x]), lambda: ops.GradClip([x], [x[:2]]), lambda: ops.GradClip([x], [f, f]), lambda: ops.GradClip([i]),
           lambda: ops.GradClip([x]).clip(-1.0), lambda: ops.GradClip([x]).clip(float("nan")), lambda: ops.GradClip([x]).clip(float("inf")), lambda: ops.GradClip([x]).norm(f)]
    for k, call in enumerate(bad):
        with pytest.raises(pkg.C6Error):
            call()
            print("not refused:", k)
    c = ops.GradClip([x])
    c.close()
    c.close()
    with pytest.raises(pkg.C6Error):
        c.norm()


def test_sizes_beyond_32_bits_are_refused():
    """their low 32 bits would be sizes that can be worked on"""
    torch, ops, _ = setup()
    one = torch.zeros(1, 1, device="cuda")
    for rows, width in ((1 << 31, 1), ((1 << 32) + 2, 1), (1, (1 << 30) + 1), (1, (1 << 32) + 5)):
        x = one.expand(rows, width)
        for call in (lambda: ops.logits_process(x, out=x), lambda: ops.policy_loss(x, torch.zeros(1, dtype=torch.int32, device="cuda"))):
            with pytest.raises(pkg.C6Error, match="2\\^30"):
                call()
    ids = torch.zeros(1, dtype=torch.int32, device="cuda").expand((1 << 32) + 3)
    with pytest.raises(pkg.C6Error, match="2\\^30"):
        ops.logits_process(one, history=ids, penalties=torch.ones(3, device="cuda"))


# ---- clipping -------------------------------------------------------------------------------------------------------------
def clip_case(torch, dts, sizes, kinds, seed, spread=4, lead=1):
    """tensors of `sizes` at odd addresses, scales apart by orders of magnitude"""
    rng = np.random.default_rng(seed)
    out = []
    for i, (k, kind) in enumerate(zip(sizes, kinds)):
        t = torch.empty(k + lead, dtype=dts[kind], device="cuda")[i % 2 * lead:][:k]
        t.copy_(torch.tensor(rng.normal(0, 10.0 ** -(i % spread), k), device="cuda"))
        out.append(t)
    return out


def clip_oracle(grads, max_norm):
    v = [host(g) for g in grads]
    norm = np.sqrt(sum(float((a * a).sum()) for a in v))
    return norm, [a * min(1.0, max_norm / (norm + 1e-6)) for a in v]


def clip_near(outs, want, kinds):
    for o, w, k in zip(outs, want, kinds):      # the factor and the product: half a step of f32 each
        po.near(host(o), w, 3 * po.E32 * np.abs(w), k, "clipped")


CLIP = [([1], ["f32"]), ([0, 3, 0], ["f32", "f16", "bf16"]), ([7, 1, 64, 1000, 33], ["f32"] * 5), ([5, 40000, 32768, 32769, 65536], ["bf16", "f32", "f16", "bf16", "f32"]),
        ([300001, 2, 99999], ["f16", "bf16", "f32"]), ([17] * 400, ["f32", "bf16"] * 200), ([3_000_001, 123457], ["bf16", "f32"])]


@pytest.mark.parametrize("i", range(len(CLIP)))
@pytest.mark.parametrize("max_norm", [0.5, 1e9, 0.0])
def test_clip(i, max_norm):
    torch, ops, dts = setup()
    sizes, kinds = CLIP[i]
    grads = clip_case(torch, dts, sizes, kinds, i)
    norm, want = clip_oracle(grads, np.float32(max_norm))
    before = [g.clone() for g in grads]
    outs = [torch.full_like(g, 3.0) for g in grads]
    c = ops.GradClip(grads, outs)
    n = c.clip(max_norm)
    assert abs(float(n) - norm) <= 2 * po.E32 * norm
    clip_near(outs, want, kinds)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    assert torch.equal(c.norm(), n)
    d = ops.GradClip(grads)
    assert torch.equal(d.norm(), n) and all(torch.equal(a, b) for a, b in zip(grads, before))
    assert torch.equal(d.clip(max_norm), n)
    assert all(torch.equal(a, b) for a, b in zip(grads, outs))      # in place: the same bits
    if max_norm > norm:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_clip_neither_overflows_nor_vanishes():
    torch, ops, _ = setup()
    for scale in (1e30, 1e-30):
        g = torch.full((100000,), scale, device="cuda")
        c = ops.GradClip([g])
        want = scale * np.sqrt(1e5)
        assert abs(float(c.norm()) - want) <= 1e-6 * want
    g = torch.full((100000,), 1e30, device="cuda")
    ops.GradClip([g]).clip(1.0)
    assert abs(float(g[7]) * np.sqrt(1e5) - 1) < 1e-6


def test_clip_of_nothing():
    torch, ops, _ = setup()
    e = torch.empty(0, device="cuda")
    c = ops.GradClip([e, e.half()])
    assert float(c.norm()) == 0 and float(c.clip(1.0)) == 0


def test_clip_infinities_and_nan():
    torch, ops, _ = setup()
    g = [torch.ones(5, device="cuda"), torch.ones(70000, dtype=torch.bfloat16, device="cuda")]
    g[1][69999] = np.inf
    o = [torch.empty_like(t) for t in g]
    assert float(ops.GradClip(g, o).clip(1.0)) == np.inf                # factor 0: the infinity becomes NaN, the rest 0
    assert bool((o[0] == 0).all()) and bool((o[1][:-1] == 0).all()) and bool(o[1][-1].isnan())
    g[0][2] = np.nan
    assert bool(ops.GradClip(g, o).clip(1.0).isnan().all()) and all(bool(t.isnan().all()) for t in o)


def test_clip_size_beyond_32_bits():
    torch, ops, _ = setup()
    n = (1 << 32) + 5
    g = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    c = ops.GradClip([g])
    want = 0.5 * np.sqrt(float(n))
    assert abs(float(c.clip(1.0)) - want) <= 1e-6 * want
    f = 0.5 / want
    assert abs(float(g[n - 1]) - f) <= f * 2.0 ** -8 and bool((g[-3:] == g[0]).all()) and bool((g[1 << 31:(1 << 31) + 9] == g[0]).all())


# ---- together, on streams, captured ---------------------------------------------------------------------------------------
def test_a_run_of_them_together():
    """a linear policy over the legal moves, one step: penalties and mask on the logits, loss and gradient, the weights' gradient, clipping -- against the
    same in float64.  The matrix products are torch's in float32: 2 n half steps of the terms' magnitudes for a sum of n."""
    torch, ops, _ = setup()
    rng = np.random.default_rng(9)
    rows, feat, width = 64, 50, 225
    h = rng.normal(0, 1, (rows, feat)).astype(np.float32)
    W = rng.normal(0, 0.3, (feat, width)).astype(np.float32)
    keep = rng.random((rows, width)) < 0.6
    keep[:, 0] = True
    t = rng.random((rows, width)).astype(np.float32) * keep
    hist = rng.integers(0, width, (rows, 20)).astype(np.int32)
    pen = np.array([1.2, 0.1, 0.2], np.float32)
    g = lambda a: torch.tensor(a, device="cuda")  # noqa: E731
    H, mask = g(h), g(po.pack(keep))
    x = H @ g(W)
    y = ops.logits_process(x, mask=mask, history=g(hist), penalties=g(pen))
    loss, lse, total, dy = ops.policy_loss(y, g(t), grad_scale=1.0 / rows)            # the mask has become -infinity
    loss2, _, _, dy2 = ops.policy_loss(y, g(t), mask=mask, grad_scale=1.0 / rows)
    assert torch.equal(loss, loss2) and torch.equal(dy, dy2)
    dW = H.t() @ dy
    c = ops.GradClip([dW])
    norm = c.clip(0.01)
    yy, ytol = po.process(host(x), po.pack(keep), history=hist, penalties=pen)
    po.near(host(y), yy, ytol, "f32", "process")
    want, tol = po.loss(host(y), t, po.pack(keep), 1.0 / rows)
    po.near(host(loss), want["loss"], tol["loss"], "f32", "loss")
    po.near(host(dy), want["grad"], tol["grad"], "f32", "gradient")
    ref = h.astype(np.float64).T @ want["grad"]
    mag = np.abs(h.astype(np.float64)).T @ (2 * rows * po.E32 * np.abs(want["grad"]) + tol["grad"])
    n = np.linalg.norm(ref)
    assert abs(float(norm) - n) <= np.linalg.norm(mag) + 2 * po.E32 * n
    f = 0.01 / (n + 1e-6)
    po.near(host(dW), ref * f, (mag + np.abs(ref) * np.linalg.norm(mag) / n) * f + 4 * po.E32 * np.abs(ref * f), "f32", "clipped")


@pytest.mark.parametrize("rows,width", [(64, 361), (2, 100003)])
def test_other_stream_and_graph(rows, width):
    """on a stream of their own, then captured: several replays on new inputs with eager work between, two graphs at once; every replay equals the eager call"""
    torch, ops, _ = setup()
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, w = new(rows, width), new(rows, width).abs()
    hist = torch.randint(0, width, (rows, 50), dtype=torch.int32, device="cuda")
    pen = torch.tensor([1.3, 0.2, 0.1], device="cuda")
    G = torch.empty(rows, width, device="cuda")
    clip = ops.GradClip([G])

    def step():
        y = ops.logits_process(x, history=hist, penalties=pen)
        loss, lse, total, g = ops.policy_loss(y, w, grad_scale=1.0, grad=G)
        b = ops.policy_loss_grad(y, w, lse, total, loss)
        return [y, loss, lse, total, b, clip.clip(0.1), G]

    want = [v.clone() for v in step()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [v.clone() for v in step()]
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        y2 = ops.logits_process(x, history=hist, penalties=pen)
        out2 = ops.policy_loss(y2, w, grad_scale=2.0)
    for k in range(4):
        x.copy_(new(rows, width))
        hist.copy_(torch.randint(0, width, (rows, 50), dtype=torch.int32, device="cuda"))
        eager = [v.clone() for v in step()]
        eager2 = ops.policy_loss(eager[0], w, grad_scale=2.0)
        G.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            second.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), k
        assert all(torch.equal(a, b) for a, b in zip(out2, eager2)), k


def test_same_bits_every_time():
    torch, ops, _ = setup()
    x = torch.randn(5, 131072, device="cuda").bfloat16()
    t = torch.rand(5, 131072, device="cuda")
    hist = torch.randint(0, 50, (5, 9000), dtype=torch.int32, device="cuda")
    pen = torch.tensor([1.1, 0.3, 0.2], device="cuda")
    first = None
    for _ in range(5):
        g = ops.policy_loss(x, t, grad_scale=1.0)
        c = ops.GradClip([g[3]])
        now = [*g, ops.logits_process(x, history=hist, penalties=pen), c.norm(), c.clip(0.01)]
        now = [v.clone() for v in now]
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
        first = now
