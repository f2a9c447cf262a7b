"""The trainer's policy targets at the ends of their range."""
import numpy as np
import pytest
import torch  # noqa: F401  (before the library is first used: they share one HIP runtime)

from gpu_common import need_gpu, pkg
from test_gpu_train_policy import batch, net, trainer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [2.0 ** 122, 2.0 ** -120])
def test_visits_of_any_size(scale):
    """finite visits whose sum exceeds the largest float (or that are next to the smallest): normalised like the same visits in ordinary numbers, bit for bit"""
    need_gpu()
    _, blob = net()
    w, p, b, q, pi = batch(9)
    pi = np.minimum(pi, 60).astype(np.float32)
    assert np.isfinite(pi * np.float32(scale)).all()
    out = []
    for s in (1.0, scale):
        t = trainer(blob)
        t.set_policy_loss(pkg.POLICY_LOSS_VISITS)
        loss = t.step(w, p, b, pi * np.float32(s))
        out.append((loss, t.gradients(), t.export_weights()))
        t.close()
    if scale > 1:
        assert ((pi * (b == 0)).astype(np.float64).sum(1).max() * scale) > np.finfo(np.float32).max
    assert out[0][0] == out[1][0] and all(np.array_equal(x, y) for x, y in zip(out[0][1:], out[1][1:]))
