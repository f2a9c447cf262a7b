"""The trainer's policy loss over the empty cells (moves or visit counts) and its gradient clipping, against PyTorch autograd in float64 on the CPU.

Tolerances: those of test_gpu_train.py's strict cases (the same forward and backward kernels; here too no ReLU input lies near 0); clipping adds the
factor's and the product's half steps of f32."""
import numpy as np
import pytest
import torch  # noqa: F401  (before the library is first used: they share one HIP runtime)

import torch_ref as tr
from gpu_common import need_gpu, pkg

pytestmark = pytest.mark.gpu
N, C, BLOCKS, B = 9, 64, 2, 8
E32 = 2.0 ** -24


def net(seed=38):
    torch.manual_seed(seed)
    m = tr.WeightedPolicy(N, C, BLOCKS)
    tr.decisive_bn(m)
    return m, tr.blob_of(m)


def batch(seed, full=None):
    w, p, b, q = tr.make_batch(N, B, seed=seed)
    rng = np.random.default_rng(seed)
    b = b.numpy()
    for i in range(B):      # a move on an empty cell for most positions, on a stone for the last
        cells = np.flatnonzero(b[i] == 0) if i < B - 1 else np.flatnonzero(b[i] != 0)
        q[i] = float(rng.choice(cells))
    if full is not None:
        b[full] = 1.0
    pi = (rng.random((B, N * N)) ** 6 * 40).astype(np.float32).round()      # some on stones too: they count for nothing
    pi[2] = 0
    return w.numpy(), p.numpy(), b, q.numpy(), pi


def reference(m, data, visits, lr):
    """(loss, gradient blob, blob after one SGD step) in float64"""
    w, p, b, q, pi = [torch.tensor(x, dtype=torch.float64) for x in data]
    m = m.double()
    m.train()
    opt = torch.optim.SGD(m.parameters(), lr=lr, momentum=0.9)
    pol, value = m(p, b)
    empty = b == 0
    t = pi * empty if visits else torch.zeros_like(b).scatter_(1, q.long()[:, None], 1.0) * empty
    if visits:
        t = t / t.sum(1, keepdim=True).clamp(min=1e-30)
    among = (pol * empty).sum(1, keepdim=True)
    logp = torch.where(empty, torch.log(pol) - torch.log(torch.where(among > 0, among, 1.0)), 0.0)
    loss = torch.mean((w - value).pow(2)) - (t * logp).sum(1).mean()
    opt.zero_grad()
    loss.backward()
    opt.step()
    return float(loss.detach()), tr.blob_of(m, grads=True), tr.blob_of(m)


def trainer(blob, **kw):
    t = pkg.Trainer(N, C, BLOCKS, B, lr=0.01, momentum=0.9, **kw)
    t.load_weights(blob)
    return t


@pytest.mark.parametrize("full", [None, 4])
@pytest.mark.parametrize("kind", [pkg.POLICY_LOSS_LEGAL, pkg.POLICY_LOSS_VISITS])
def test_loss_over_the_empty_cells(kind, full):
    need_gpu()
    m, blob = net()
    data = batch(7, full)
    assert tr.relu_margin(m, [torch.tensor(x) for x in data[:4]]) > 2e-4
    t = trainer(blob)
    t.set_policy_loss(kind)
    w, p, b, q, pi = data
    target = pi if kind == pkg.POLICY_LOSS_VISITS else q
    alone = t.loss(w, p, b, target)
    loss = t.step(w, p, b, target)
    grads, after = t.gradients(), t.export_weights()
    t.close()
    ref_loss, ref_grads, ref_after = reference(m, data, kind == pkg.POLICY_LOSS_VISITS, 0.01)
    assert alone == loss and abs(loss - ref_loss) <= 1e-4 * max(1.0, abs(ref_loss))
    assert np.linalg.norm(grads - ref_grads) <= 1e-4 * np.linalg.norm(ref_grads)
    off = 0
    for s, isp in tr._tensors(m):
        k = s.numel()
        for got, want in ((grads, ref_grads), (after, ref_after)):
            g, r = got[off:off + k], want[off:off + k]
            if isp:      # (loss() has moved the running statistics once more)
                assert np.abs(g - r).max() <= 1e-3 * max(np.abs(r).max(), 1e-6) + 1e-6, (off, k)
        off += k


def test_the_default_is_as_it_was():
    """bit for bit: a trainer that never heard of the new losses, and one that went through them and back"""
    need_gpu()
    _, blob = net()
    w, p, b, q, pi = batch(3)
    outs = []
    for touched in (False, True):
        t = trainer(blob)
        if touched:
            t.set_policy_loss(pkg.POLICY_LOSS_VISITS)
            t.set_policy_loss(pkg.POLICY_LOSS_REFERENCE)
            t.set_clip(1.0)
            t.set_clip(None)
        losses = [t.step(w, p, b, q) for _ in range(2)]
        outs.append((losses, t.gradients(), t.export_weights()))
        t.close()
    assert outs[0][0] == outs[1][0] and all(np.array_equal(x, y) for x, y in zip(outs[0][1:], outs[1][1:]))


def test_clipping():
    need_gpu()
    _, blob = net()
    w, p, b, q, pi = batch(5)
    t = trainer(blob)
    t.step(w, p, b, q)
    plain = t.gradients().astype(np.float64)
    norm = np.linalg.norm(plain)
    t.close()
    for max_norm in (0.1 * norm, 10.0 * norm, 0.0):
        t = trainer(blob)
        t.set_clip(max_norm)
        t.step(w, p, b, q)
        f = min(1.0, np.float32(max_norm) / (norm + 1e-6))
        got = t.gradients()
        assert abs(t.grad_norm() - norm) <= 2 * E32 * norm
        assert (np.abs(got - plain * f) <= 4 * E32 * np.abs(plain * f) + 2.0 ** -126).all()
        if f == 1.0:
            assert np.array_equal(got, plain.astype(np.float32))
        # the first step of SGD: p - lr * g, the running statistics aside (no gradient there)
        after = t.export_weights()
        moved = np.flatnonzero(plain != 0)
        want = blob[moved].astype(np.float64) - np.float32(0.01) * got[moved].astype(np.float64)
        assert (np.abs(after[moved] - want) <= 3 * E32 * (np.abs(blob[moved]) + np.abs(want))).all()
        t.set_clip(None)
        t.step(w, p, b, q)
        with pytest.raises(pkg.C6Error, match="not clipped"):
            t.grad_norm()
        t.close()


def test_visits_from_the_replay_buffer():
    """step_replay draws what sample(want_pi=True) draws, and trains on it as step does, bit for bit"""
    need_gpu()
    _, blob = net()
    rng = np.random.default_rng(2)
    games = []
    for _ in range(3):
        board, path, pis = np.zeros((N, N), np.int8), [], []
        for k in range(12):
            r, c = [int(x) for x in rng.choice(np.argwhere(board == 0))]
            path.append((-1 if k % 2 else 1, board.copy(), (r, c)))
            pis.append(rng.integers(0, 50, N * N) * (board.reshape(-1) == 0))
            board[r, c] = -1 if k % 2 else 1
        games.append((1, path, pis))
    rb = pkg.ReplayBuffer(N, 100)
    rb.push_records(pkg.encode_tuples(N, games))
    w, p, b, q, pi = rb.sample(B, seed=11, draw_id=4, want_pi=True)
    assert pi.sum() > 0
    out = []
    for replay in (True, False):
        t = trainer(blob)
        t.set_policy_loss(pkg.POLICY_LOSS_VISITS)
        t.set_clip(0.5)
        loss = t.step_replay(rb, seed=11, draw_id=4) if replay else t.step(w, p, b, pi)
        out.append((loss, t.grad_norm(), t.export_weights()))
        t.close()
    rb.close()
    assert out[0][:2] == out[1][:2] and np.array_equal(out[0][2], out[1][2])


def test_refusals():
    need_gpu()
    _, blob = net()
    w, p, b, q, pi = batch(1)
    t = trainer(blob)
    for call in (lambda: t.set_policy_loss(3), lambda: t.set_policy_loss(-1), lambda: t.set_clip(float("nan")), lambda: t.set_clip(float("inf")), lambda: t.grad_norm(),
                 lambda: t.step(w, p, b, pi)):
        with pytest.raises(pkg.C6Error):
            call()
    t.set_policy_loss(pkg.POLICY_LOSS_VISITS)
    for bad in (-1.0, np.nan, np.inf):
        v = pi.copy()
        v[3, 5] = bad
        with pytest.raises(pkg.C6Error):
            t.step(w, p, b, v)
    with pytest.raises(pkg.C6Error):
        t.step(w, p, b, q)
    assert np.isfinite(t.step(w, p, b, pi))
    t.close()
