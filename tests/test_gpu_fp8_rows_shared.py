"""8-bit rows as a program has them beside other work: calls of several threads on one
context, batches whose buffers hold NaN wherever nothing is listed."""
import threading

import numpy as np
import pytest
import torch

import wohper_amd as wa
from test_gpu_fp8_rows import Layer, Step, f64, ordered_ctx  # noqa: F401
from test_gpu_fp8_rows_tiles import TALL, TILE, Case, check, plan

pytestmark = pytest.mark.gpu


def test_threads_of_one_context(ctx):
    """Products that use the context's parts and counters, from two threads: each call's
    launches stay together, so both have their own results."""
    sizes = [(128, 4096, 4096, TILE), (5000, 4112, 4096, TALL)]
    jobs = []
    for i, (n, rows, cols, kind) in enumerate(sizes):
        p = plan(n, rows, cols)
        assert p[0] == kind and (p[1] > 1 if kind == TILE else p[3] > p[2])
        c = Case(ctx.raw, i, n, rows, cols)
        jobs.append((c, n, rows, [torch.zeros(n, rows, dtype=torch.bfloat16, device="cuda") for _ in range(20)]))
    torch.cuda.synchronize()

    def run(c, n, rows, ys):
        for y in ys:
            ctx.raw.fp8_rows_mm_async(c.h, 0, rows, c.rows.c, n, y.data_ptr(), rows, True)

    threads = [threading.Thread(target=run, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    ctx.raw.synchronize()
    for c, n, rows, ys in jobs:
        check(ys[0], c.x(), c.w(0, rows), c.cols)
        assert all(torch.equal(y, ys[0]) for y in ys)
        c.close()


@pytest.mark.parametrize("npos", [3, 40, 300])
@pytest.mark.parametrize("bf16", [False, True])
def test_a_padded_layer_reads_nothing_that_is_not_listed(ctx, npos, bf16):
    """Half of the positions are padding with NaN inputs, and every buffer of the step is
    full of NaN before it: the other positions' sums are those of clean buffers."""
    rng = np.random.default_rng(npos)
    layer = Layer(ctx, rng, 6, 512, 256)
    outs = []
    for dirty in (False, True):
        step = Step(layer, npos, 2, bf16)
        step.fill(npos)
        pad = slice(npos - npos // 2, npos)
        step.ids[pad] = -1
        if dirty:
            step.x[pad] = float("nan")
            step.weights[pad] = float("nan")
            for t in (step.gu, step.y, step.out):
                t.fill_(float("nan"))
            for t in (step.x8, step.h8):
                t.codes.fill_(0x7F)
                t.scales.fill_(255)
        step.run(ctx)
        ctx.synchronize()
        assert bool((step.out[pad] == 0).all())
        outs.append(step.out.clone())
    assert torch.equal(outs[0], outs[1]) and np.isfinite(f64(outs[0])).all() and float(outs[0].abs().max()) > 0
    layer.close()


def test_a_graph_serves_batches_of_every_fill(ctx):
    """One captured step, replayed with no position, one, and all of them listed."""
    rng = np.random.default_rng(3)
    layer = Layer(ctx, rng, 6, 512, 256)
    step = Step(layer, 600, 4, True)
    step.fill(0)
    step.run(ctx)
    ctx.synchronize()
    g = ctx.capture(lambda: step.run(ctx))
    for seed, used in ((1, 0), (2, 1), (3, 600), (4, 0), (5, 77)):
        step.fill(seed)
        step.ids[used:] = -1
        step.run(ctx)
        ctx.synchronize()
        eager = step.out.clone()
        step.out.fill_(float("nan"))
        step.y.fill_(float("nan"))
        torch.cuda.synchronize()
        ctx.graph_launch(g)
        ctx.synchronize()
        assert torch.equal(step.out, eager) and bool((eager[used:] == 0).all())
        assert used == 0 or float(eager[:used].abs().max()) > 0
    ctx.graph_release(g)
    layer.close()


def test_a_capture_that_needs_more_memory_fails_and_leaves_the_context():
    """A product whose parts, or a plan whose counts, do not fit what the context has: the
    capture ends in an error, is never launched, and eager calls go on."""
    fresh = wa.Context(0)
    sizes = [(128, 1024, 4096), (128, 4096, 4096)]
    assert all(plan(*s)[0] == TILE and plan(*s)[1] > 1 for s in sizes)
    cases = [Case(fresh, i, *s) for i, s in enumerate(sizes)]
    ys = [torch.zeros(n, rows, dtype=torch.bfloat16, device="cuda") for n, rows, _ in sizes]
    ids = torch.randint(0, 64, (20000,), dtype=torch.int32, device="cuda")
    out = [torch.zeros(k, dtype=torch.int32, device="cuda") for k in (65, 20000, 20000)]
    torch.cuda.synchronize()

    def product(i):
        fresh.fp8_rows_mm_async(cases[i].h, 0, sizes[i][1], cases[i].rows.c, sizes[i][0], ys[i].data_ptr(), sizes[i][1], True)

    def lists_of():
        fresh.expert_plan_async(ids.data_ptr(), 20000, 1, 64, out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr())

    for calls in ((lists_of,), (lambda: product(0),)):
        with pytest.raises(wa.DeepSeekV4KernelError):
            fresh.graph_capture(lambda calls=calls: [c() for c in calls])
    product(0)
    fresh.synchronize()
    with pytest.raises(wa.DeepSeekV4KernelError):
        fresh.graph_capture(lambda: (product(0), product(1)))
    lists_of()
    for i in range(2):
        product(i)
    fresh.synchronize()
    for i, (n, rows, cols) in enumerate(sizes):
        check(ys[i], cases[i].x(), cases[i].w(0, rows), cols)
    assert torch.equal(torch.bincount(ids, minlength=64).cumsum(0), out[0][1:].long())
    g = fresh.graph_capture(lambda: (product(0), product(1), lists_of()))
    for _ in range(3):
        for t in ys + out:
            t.fill_(3)
        torch.cuda.synchronize()
        fresh.graph_launch(g)
        fresh.synchronize()
        for i, (n, rows, cols) in enumerate(sizes):
            check(ys[i], cases[i].x(), cases[i].w(0, rows), cols)
        assert torch.equal(torch.bincount(ids, minlength=64).cumsum(0), out[0][1:].long())
    fresh.graph_release(g)
    for c in cases:
        c.close()
    fresh.close()
