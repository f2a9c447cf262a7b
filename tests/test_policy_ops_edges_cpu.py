"""Edges of the operators on logits and gradients without a GPU: outputs that overlap what a call reads are refused before a device is looked for, and interleaved or
neighbouring memory is not."""
import pytest

from test_policy_ops_cpu import A, BAD, NO_GPU, grad_of, logits, loss, pkg, process

# logits: 4 rows of 10 f32 from A on, 40 bytes a row; the output of process and grad_of from 4 A on, 40 bytes a row
OUT = 4 * A
HIST = dict(history=8 * A, hs=5, n=9 * A, cap=5, pen=10 * A, ps=3)


@pytest.mark.parametrize("call,kw", [
    (process, dict(bias=OUT, bs=10)), (process, dict(bias=OUT + 156)), (process, dict(bias=OUT - 36)), (process, dict(bias=OUT - 120, bs=10)), (process, {**HIST, "history": OUT + 4}), (process, {**HIST, "n": OUT + 144}),
    (process, {**HIST, "n": OUT - 12}), (process, {**HIST, "pen": OUT - 8}), (process, {**HIST, "pen": OUT + 156, "ps": 0}), (process, {**HIST, "history": OUT - 4 * 15 - 4 * 4}),
    (grad_of, dict(target=OUT, kind=2, ts=10)), (grad_of, dict(target=OUT + 8, kind=2, ts=10)), (grad_of, dict(target=OUT + 156)), (grad_of, dict(target=OUT - 24, kind=1)), (grad_of, dict(lse=OUT)),
    (grad_of, dict(total=OUT + 144)), (grad_of, dict(dloss=OUT + 100)), (grad_of, dict(dloss=OUT - 12, ds=1)),
    (loss, dict(grad=OUT, gs=10, target=OUT, kind=2, ts=10)), (loss, dict(grad=OUT, gs=10, target=OUT + 40)), (loss, dict(grad=OUT, gs=10, stats=OUT + 120)), (loss, dict(stats=A + 8)), (loss, dict(stats=A - 12)),
    (loss, dict(stats=2 * A, kind=2, ts=10)), (loss, dict(stats=2 * A + 4, kind=0))])
def test_outputs_that_overlap_an_argument(call, kw):
    assert call(logits(), **kw) == BAD
    assert b"overlaps" in pkg.lib().c6_last_error()


@pytest.mark.parametrize("mask", [dict(mask=OUT, mask_row=2, mask_byte=1), dict(mask=OUT + 159, mask_row=0, mask_byte=1), dict(mask=OUT - 7, mask_row=1, mask_byte=4), dict(mask=OUT + 100, mask_row=1, mask_byte=4)])
def test_outputs_that_overlap_the_mask(mask):
    assert process(logits(**mask)) == BAD and grad_of(logits(**mask)) == BAD and loss(logits(**mask), grad=OUT, gs=10) == BAD


def test_neighbours_and_interleaved_rows_are_not_refused():
    if pkg.device_count() > 0:
        pytest.skip("a GPU is present: the addresses are not real")
    near = [(process, logits(), dict(bias=OUT + 160, bs=10)), (process, logits(), dict(bias=OUT - 40)), (process, logits(), {**HIST, "history": OUT + 160, "n": OUT - 16, "pen": OUT - 16 - 48}),
            (grad_of, logits(), dict(target=OUT + 160, kind=2, ts=10, lse=OUT - 16, total=OUT - 32, dloss=OUT - 48, ds=1)), (loss, logits(), dict(grad=OUT, gs=10, stats=OUT + 160)),
            # columns of one buffer, 30 floats a row: logits, weights or biases, the output
            (process, logits(x_stride=30), dict(bias=A + 40, bs=30, out=A + 80, os=30)), (grad_of, logits(x_stride=30), dict(target=A + 40, kind=2, ts=30, grad=A + 80, gs=30)),
            (loss, logits(x_stride=30), dict(target=A + 80, kind=2, ts=30, grad=A + 40, gs=30)), (loss, logits(x_stride=30), dict(target=A + 80, kind=2, ts=30, grad=A, gs=30)),
            # one bias, one mask for all rows behind a row of the output
            (process, logits(x_stride=30), dict(bias=OUT + 80, bs=0, out=OUT, os=30)), (process, logits(x_stride=30, mask=OUT + 80, mask_row=120, mask_byte=1), dict(out=OUT, os=30)),
            (process, logits(mask=OUT - 8, mask_row=1, mask_byte=4), {}), (process, logits(mask=OUT + 160, mask_row=2, mask_byte=1), {})]
    for k, (call, l, kw) in enumerate(near):
        assert call(l, **kw) == NO_GPU, (k, pkg.lib().c6_last_error())


@pytest.mark.parametrize("kw", [dict(mask=16 * A, mask_row=1 << 62, mask_byte=1), dict(mask=16 * A, mask_row=0, mask_byte=1 << 62), dict(mask=16 * A, mask_row=1 << 61, mask_byte=1 << 61)])
def test_masks_beyond_the_address_space(kw):
    assert process(logits(**kw)) == BAD and loss(logits(**kw)) == BAD and grad_of(logits(**kw)) == BAD


def test_strides_beyond_the_address_space():
    assert grad_of(logits(), ds=1 << 62) == BAD
    if pkg.device_count() == 0:      # strides of what is not there are not looked at
        assert process(logits(), hs=1 << 62, ps=1 << 62, bs=1 << 62) == NO_GPU and loss(logits(), gs=1 << 62) == NO_GPU
