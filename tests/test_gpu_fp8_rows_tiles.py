"""Products of 8-bit rows on tiles of 128 x 256 and 256 x 256, whose workgroups take
tiles from shared counters: grouped by expert, gathered, with rows that are none or
NaN, odd counts of blocks and more than a chunk of scales (64 blocks), launches one
behind another, in graphs and from two contexts.  Each case asserts the kernel that its
sizes are meant for, so that another rule moves no test to another kernel unseen.

Tolerances as in test_gpu_fp8_rows: bf16 products are within 2^-10 of sum |w||x| (eight
products aligned to the largest) and half a step of bf16, 2^-8."""
import ctypes
import threading

import numpy as np
import pytest
import torch

import wohper_amd as wa
from test_gpu_fp8_rows import BLOCK, COLUMN, NONE, E4M3, Rows, gpu_near, i32, lists, ordered_ctx  # noqa: F401

pytestmark = pytest.mark.gpu
THIN, TILE, HALF, TALL = 1, 2, 3, 4


def plan(n, rows, cols, groups=0, bf16=True, f32=False, special=False):
    """Kernel, ranges, workgroups and most tiles of a product (groups 0: without lists)."""
    p = (ctypes.c_uint64 * 4)()
    status = wa.load_library().wh_debug_fp8_rows_plan(n, max(groups, 1), int(groups > 0), rows, cols, int(f32), int(special),
                                                      int(bf16), p)
    assert status == 0
    return tuple(p)


class Case:
    """Random rows and a random UE8M0 weight, made on the GPU; f64 values of either by ranges."""

    def __init__(self, ctx, seed, n, rows, cols):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.ctx, self.cols, self.table = ctx, cols, torch.from_numpy(E4M3).cuda()
        self.codes, self.x_codes = (torch.randint(0, 256, (m, cols), generator=g, device="cuda", dtype=torch.uint8)
                                    for m in (rows, n))
        for c in (self.codes, self.x_codes):  # neither +-480 nor NaN
            c[(c & 0x7F) == 0x7F] ^= 1
        self.scales = torch.randint(117, 124, (rows // 16, cols // BLOCK), generator=g, device="cuda", dtype=torch.uint8)
        self.x_scales = torch.randint(115, 126, (n, cols // BLOCK), generator=g, device="cuda", dtype=torch.uint8)
        self.rows = Rows(n, cols)
        self.put()
        torch.cuda.synchronize()
        self.h = ctx.store_fp8_device(self.codes.data_ptr(), rows, cols, self.scales.data_ptr(), *self.scales.shape)

    def put(self):
        n = self.x_codes.shape[0]
        order = torch.from_numpy(COLUMN).cuda()
        self.rows.codes.copy_(self.x_codes.reshape(n, -1, BLOCK)[:, :, order].reshape(n, self.cols))
        self.rows.scales[:, :self.cols // BLOCK] = self.x_scales

    def w(self, a, b):
        s = torch.exp2(self.scales[a // 16:-(-b // 16)].double() - 127)
        return self.table[self.codes[a:b].int()] * s.repeat_interleave(16, 0)[a % 16:a % 16 + b - a].repeat_interleave(BLOCK, 1)

    def x(self):
        nan = self.table.clone()
        nan[[0x7F, 0xFF]] = float("nan")
        s = torch.where(self.x_scales == 255, float("nan"), torch.exp2(self.x_scales.double() - 127))
        return nan[self.x_codes.int()] * s.repeat_interleave(BLOCK, 1)

    def close(self):
        self.ctx.release(self.h)


def check(y, x, w, cols):
    """y [m, rows] of x rows: NaN where a row has NaN, else the products."""
    bad = torch.isnan(x).any(1)
    assert bool(torch.isnan(y[bad]).all()) and not bool(torch.isnan(y[~bad]).any())
    gpu_near(y[~bad], x[~bad], w, True, cols)


@pytest.mark.parametrize("kind,n_groups,n,rows,cols", [
    (TALL, 64, 24000, 4096, 4096), (TALL, 64, 16000, 4096, 4224), (TALL, 20, 16000, 4096, 8320), (TALL, 64, 20000, 4112, 4096),
    (HALF, 64, 4000, 1024, 4096), (HALF, 64, 1500, 1024, 4096), (HALF, 64, 3000, 1024, 8320), (HALF, 64, 4000, 1024, 4224)])
@pytest.mark.parametrize("gather", [True, False])
def test_groups_on_large_tiles(ctx, kind, n_groups, n, rows, cols, gather):
    assert plan(n, rows, cols, n_groups)[0] == kind
    rng = np.random.default_rng(n)
    n_x = 900 if gather else n
    c = Case(ctx, n, n_x, n_groups * rows, cols)
    starts = lists(rng, n_groups, n, "ragged")
    tile = 256 if kind == TALL else 128
    assert kind != TALL or sum(-(-m // tile) for m in np.diff(starts)) * -(-rows // 256) > 256  # the counters are asked
    at = rng.integers(0, n_x, n) if gather else np.arange(n)
    if gather:
        at[rng.integers(0, n, 20)] = NONE
        at[rng.integers(0, n, 20)] = n_x
    hit = at[[int(starts[-1]) // 2, int(starts[-1]) - 1, 3]] % n_x  # NaN in rows that are listed
    hit = hit[hit < n_x]
    c.x_codes[hit[0], cols - 1] = 0x7F
    c.x_scales[hit[1], 0] = 255
    c.x_codes[hit[-1], 77] = 0xFF
    c.put()
    s, r = i32(starts), i32(at)
    y = torch.full((n + 1, rows + 3), 5.0, dtype=torch.bfloat16, device="cuda")
    for _ in range(2):
        ctx.fp8_rows_mm_groups_async(c.h, 0, rows, n_groups, c.rows.c, n_x, r.data_ptr() if gather else None, s.data_ptr(), n,
                                     y.data_ptr(), rows + 3, True)
    ctx.synchronize()
    assert bool((y[starts[-1]:] == 5.0).all()) and bool((y[:, rows:] == 5.0).all())
    x, at_dev = c.x(), torch.from_numpy(at).cuda()
    for g in range(n_groups):
        a, b = int(starts[g]), int(starts[g + 1])
        if b > a:
            take = at_dev[a:b]
            none = take >= n_x
            assert bool((y[a:b, :rows][none] == 0).all())
            v = torch.where(none[:, None], 0.0, x[take.clamp(max=n_x - 1)])
            check(y[a:b, :rows], v, c.w(g * rows, (g + 1) * rows), cols)
    c.close()


@pytest.mark.parametrize("kind,n,rows,cols", [(TALL, 5000, 4112, 4096), (TALL, 4300, 4112, 4224), (TALL, 4099, 4096, 8320),
                                              (HALF, 2048, 4096, 4096), (HALF, 1500, 4096, 8320), (HALF, 2000, 4090, 4224)])
def test_nan_rows_on_large_tiles(ctx, kind, n, rows, cols):
    assert plan(n, rows, cols)[0] == kind
    c = Case(ctx, n, n, -(-rows // 16) * 16, cols)
    c.x_codes[[0, 130, n - 1], [0, 200, cols - 1]] = 0x7F
    c.x_scales[[65, n - 2], [cols // BLOCK - 1, 0]] = 255
    c.put()
    y = torch.full((n + 1, rows), 5.0, dtype=torch.bfloat16, device="cuda")
    ctx.fp8_rows_mm_async(c.h, 0, rows, c.rows.c, n, y.data_ptr(), rows, True)
    ctx.synchronize()
    assert bool((y[n] == 5.0).all())
    check(y[:n], c.x(), c.w(0, rows), cols)
    c.close()


class Counted:
    """A product whose workgroups ask the counters: more tiles than workgroups."""

    def __init__(self, ctx, seed, n, rows, cols, kind):
        p = plan(n, rows, cols)
        assert p[0] == kind and p[3] > p[2] == 256
        self.ctx, self.n, self.rows, self.cols = ctx, n, rows, cols
        self.case = Case(ctx, seed, n, rows, cols)
        self.y = torch.zeros(n, rows, dtype=torch.bfloat16, device="cuda")
        torch.cuda.synchronize()

    def run(self, y=None):
        self.ctx.fp8_rows_mm_async(self.case.h, 0, self.rows, self.case.rows.c, self.n, (self.y if y is None else y).data_ptr(),
                                   self.rows, True)

    def first(self):
        """The result, held against 64 bits."""
        self.run()
        self.ctx.synchronize()
        check(self.y, self.case.x(), self.case.w(0, self.rows), self.cols)
        return self.y.clone()


SIZES = [(5000, 4112, 4096, TALL), (1900, 5136, 8320, HALF), (4300, 4112, 8576, TALL)]


def test_counters_are_free_behind_every_launch(ctx):
    """Launches one behind another, eager and replayed, alone and in turn: each does every
    tile, so none finds the counters as another left them."""
    jobs = [Counted(ctx, i, *s) for i, s in enumerate(SIZES)]
    want = [j.first() for j in jobs]
    graphs = [ctx.capture(lambda a=a, b=b: (jobs[a].run(), jobs[b].run())) for a, b in ((0, 1), (1, 2), (2, 0))]
    for turn in range(6):
        for j in jobs:
            j.y.fill_(7.0)
        torch.cuda.synchronize()
        ctx.graph_launch(graphs[turn % 3])
        jobs[turn % 3].run()
        jobs[(turn + 2) % 3].run()
        jobs[(turn + 1) % 3].run()
        ctx.synchronize()
        assert all(torch.equal(j.y, w) for j, w in zip(jobs, want))
        for j in jobs:
            j.y.fill_(9.0)
        torch.cuda.synchronize()
        for g in graphs:
            ctx.graph_launch(g)
        ctx.synchronize()
        assert all(torch.equal(j.y, w) for j, w in zip(jobs, want))
    for g in graphs:
        ctx.graph_release(g)
    for j in jobs:
        j.case.close()


def test_counters_of_two_contexts(ctx):
    other = wa.Context(0)
    jobs = [Counted(k, i, *SIZES[0]) for i, k in enumerate((ctx.raw, other))]
    want = [j.first() for j in jobs]
    ys = [[torch.zeros_like(j.y) for _ in range(12)] for j in jobs]
    torch.cuda.synchronize()

    def run(j, out):
        for y in out:
            j.run(y)
        j.ctx.synchronize()

    threads = [threading.Thread(target=run, args=a) for a in zip(jobs, ys)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for j, w, out in zip(jobs, want, ys):
        assert all(torch.equal(y, w) for y in out)
        j.case.close()
    other.close()


@pytest.mark.parametrize("kind,n_groups,n,rows,cols,bf16", [
    (THIN, 64, 1000, 256, 640, True), (THIN, 64, 1000, 256, 640, False), (TILE, 16, 3000, 272, 8448, True),
    (TILE, 16, 3000, 272, 8448, False), (TILE, 64, 6000, 512, 1152, True), (HALF, 64, 4000, 1024, 4096, True),
    (TALL, 64, 16000, 4096, 4096, True)])
def test_results_do_not_depend_on_how_rows_are_spread(ctx, kind, n_groups, n, rows, cols, bf16):
    """The same x row in every list, over lists of all lengths: the same bits, whichever
    tile, place in it and number of rows beside it."""
    assert plan(n, rows, cols, n_groups, bf16=bf16)[0] == kind
    c = Case(ctx, n, 40, n_groups * rows, cols)
    rng = np.random.default_rng(n)
    first = {}
    for spread in range(3):
        starts = lists(rng, n_groups, n, ("ragged", "even", "one")[spread])
        at = rng.integers(0, 40, n)
        at[rng.integers(0, n, n // 2)] = 7
        s, r = i32(starts), i32(at)
        y = torch.zeros(n, rows, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
        ctx.fp8_rows_mm_groups_async(c.h, 0, rows, n_groups, c.rows.c, 40, r.data_ptr(), s.data_ptr(), n, y.data_ptr(), rows, bf16)
        ctx.synchronize()
        at_dev = torch.from_numpy(at).cuda()
        for g in range(n_groups):
            a, b = int(starts[g]), int(starts[g + 1])
            sevens = y[a:b][at_dev[a:b] == 7]
            if len(sevens):
                assert torch.equal(sevens, first.setdefault(g, sevens[0]).expand_as(sevens))
    assert len(first) == n_groups
    c.close()


@pytest.mark.parametrize("kind,n,rows", [(TALL, 16000, 4096), (HALF, 4000, 1024)])
def test_starts_that_do_not_ascend_leave_counters_and_neighbours(ctx, kind, n, rows):
    """Lists that overlap count rows more than once: the n rows of y are undefined, those
    behind them stay, and the next call finds the counters at 0."""
    n_groups, cols = 64, 4096
    assert plan(n, rows, cols, n_groups)[0] == kind
    c = Case(ctx, n, 300, n_groups * rows, cols)
    rng = np.random.default_rng(n)
    at = rng.integers(0, 300, n)
    r, y = i32(at), torch.full((n + 300, rows), 5.0, dtype=torch.bfloat16, device="cuda")
    good = lists(rng, n_groups, n, "ragged")
    for starts in ([0, n] * 32 + [0], [n, 0] * 32 + [n], list(range(0, 4000000000, 61000000))[:65], good[::-1].copy(), good):
        s = i32(starts)
        ctx.fp8_rows_mm_groups_async(c.h, 0, rows, n_groups, c.rows.c, 300, r.data_ptr(), s.data_ptr(), n, y.data_ptr(), rows, True)
        ctx.synchronize()
        assert bool((y[n:] == 5.0).all())
    x, at_dev = c.x(), torch.from_numpy(at).cuda()
    for g in range(n_groups):
        a, b = int(good[g]), int(good[g + 1])
        if b > a:
            check(y[a:b], x[at_dev[a:b]], c.w(g * rows, (g + 1) * rows), cols)
    c.close()


@pytest.mark.parametrize("kind,n_groups,n,rows,cols,bf16,special", [
    (0, 5, 200, 256, 384, True, True), (THIN, 8, 100, 256, 640, True, False), (THIN, 1, 20, 8192, 4096, True, False),
    (TILE, 16, 3000, 272, 8448, True, False), (TILE, 16, 3000, 272, 8448, False, False), (TILE, 1, 700, 4090, 1152, False, False),
    (HALF, 64, 4000, 1024, 4096, True, False), (TALL, 64, 16000, 4096, 4096, True, False)])
def test_lists_that_begin_behind_the_first_row(ctx, kind, n_groups, n, rows, cols, bf16, special):
    """Some of a longer plan's experts: starts begin and end inside y, whose other rows stay."""
    assert plan(n, rows, cols, n_groups, bf16=bf16, special=special)[0] == kind
    total = -(-n_groups * rows // 16) * 16
    c = Case(ctx, n, n, total, cols)
    if special:
        ctx.release(c.h)
        c.codes[3, 3] = 0x7F
        torch.cuda.synchronize()
        c.h = ctx.store_fp8_device(c.codes.data_ptr(), total, cols, c.scales.data_ptr(), *c.scales.shape)
    starts = n // 5 + lists(np.random.default_rng(n), n_groups, n // 2, "ragged")
    s = i32(starts)
    y = torch.full((n + 1, rows), 5.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    ctx.fp8_rows_mm_groups_async(c.h, 0, rows, n_groups, c.rows.c, n, None, s.data_ptr(), n, y.data_ptr(), rows, bf16)
    ctx.synchronize()
    assert bool((y[:starts[0]] == 5.0).all()) and bool((y[starts[-1]:] == 5.0).all())
    x = c.x()
    for g in range(n_groups):
        a, b = int(starts[g]), int(starts[g + 1])
        if b > a:
            gpu_near(y[a:b], x[a:b], c.w(g * rows, (g + 1) * rows), bf16, cols)
    c.close()
