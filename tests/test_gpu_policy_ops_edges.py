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
