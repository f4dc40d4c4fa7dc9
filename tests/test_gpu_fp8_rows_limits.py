"""8-bit rows at the ends of what their calls take: sizes that pass a launch's threads,
many routes, bf16 results where every error is as large as it can be.  Other tolerances
as in test_gpu_fp8_rows."""
import time

import numpy as np
import pytest
import torch

import wohper_amd as wa
from test_gpu_fp8_rows import BLOCK, COLUMN, E4M3, Rows, gpu_near, ordered_ctx  # noqa: F401
from test_gpu_fp8_rows_tiles import HALF, TALL, THIN, TILE, Case, plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("special", [False, True])
def test_products_of_more_outputs_than_a_launch_has_threads(ctx, special):
    """65600 x 65552 outputs.  With a code of +-480 in the weight the vector kernel does
    them, 16 x 16 a workgroup: more than 2^24 of them."""
    n, rows, cols = 65600, 65552, 128
    c = Case(ctx, 1, n, rows, cols)
    if special:
        ctx.release(c.h)
        c.codes[rows - 1, 5], c.codes[40000, 127] = 0x7F, 0xFF
        torch.cuda.synchronize()
        c.h = ctx.store_fp8_device(c.codes.data_ptr(), rows, cols, c.scales.data_ptr(), *c.scales.shape)
    y = torch.full((n + 1, rows), 5.0, dtype=torch.bfloat16, device="cuda")
    ctx.fp8_rows_mm_async(c.h, 0, rows, c.rows.c, n, y.data_ptr(), rows, True)
    ctx.synchronize()
    assert bool((y[n] == 5.0).all())
    x, w = c.x(), c.w(0, rows)
    for a, b in ((0, 300), (n // 2, n // 2 + 17), (n - 1000, n)):
        gpu_near(y[a:b], x[a:b], w, True, cols)
    for a, b in ((0, 20), (40000, 40001), (rows - 17, rows)):
        gpu_near(y[:n, a:b], x, w[a:b], True, cols)
    c.close()


def codes_of(v):
    return torch.from_numpy(np.asarray(v, np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


@pytest.mark.parametrize("kind,n,rows,cols", [
    (THIN, 3, 4096, 4096), (THIN, 3, 4096, 8192), (TILE, 3, 4096, 40704), (TILE, 700, 4096, 8192), (TILE, 600, 8192, 40704),
    (HALF, 2000, 4096, 4096), (HALF, 2000, 4096, 40704), (TALL, 4300, 4112, 4096), (TALL, 4300, 4112, 40704)])
def test_bf16_products_that_lose_most(ctx, kind, n, rows, cols):
    """Eight bytes side by side are a group.  In the first block and, with the other sign,
    the last one, each group has a product of 2^16 and seven of 7.875, which lie more than
    13 bits under it; groups between sum up to less than half a step of the f32 sum so far,
    2^20.  So everything that does not cancel may be lost: 7 * 2^-13 of S = sum |w||x| by the
    alignment, and by cols / 8 additions to an f32 sum, at most 2^-23 of S each, cols *
    2^-26; the header says 2^-10 for the first.  Then half a step of bf16, 2^-8."""
    assert plan(n, rows, cols)[0] == kind
    w, x = np.full(cols, 1.125 / 16), np.full(cols, 1.75 / 16)
    for at, sign in ((slice(0, BLOCK), 1), (slice(cols - BLOCK, cols), -1)):
        w[at], x[at] = 2.25, 3.5
        w[at][::8], x[at][::8] = sign * 256, 256
    wc, xc = codes_of(w), codes_of(x)  # by bytes
    p = E4M3[wc] * E4M3[xc]
    want, size = p.sum(), np.abs(p).sum()
    in_columns = np.empty(cols, np.uint8)
    in_columns.reshape(-1, BLOCK)[:, COLUMN] = wc.reshape(-1, BLOCK)
    h = ctx.store_fp8(np.repeat(in_columns[None], rows, 0), rows, cols, np.full((rows // 16, cols // BLOCK), 127, np.uint8),
                      rows // 16, cols // BLOCK)
    r = Rows(n, cols)
    r.codes[:, :cols] = torch.from_numpy(xc).cuda()
    r.scales[:, :cols // BLOCK] = 127
    for bf16 in (True, False):
        y = torch.empty(n, rows, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
        ctx.fp8_rows_mm_async(h, 0, rows, r.c, n, y.data_ptr(), rows, bf16)
        ctx.synchronize()
        err = float((y.double() - want).abs().max())
        bound = (2.0 ** -10 + cols * 2.0 ** -26) * size + 2.0 ** -8 * abs(want) if bf16 else (cols + 8) * 2.0 ** -24 * size
        print(f"{kind} {cols} {'bf16' if bf16 else 'f32'}: {err / size * 1024:.4f} of 2^-10 S, bound {bound / size * 1024:.4f}")
        assert err <= bound
    ctx.release(h)


class Routes:
    """Random routes, an eighth of them to no expert, and a plan's buffers."""

    def __init__(self, npos, topk, n_experts, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.npos, self.topk, self.n_experts, n = npos, topk, n_experts, npos * topk
        self.ids = torch.randint(0, n_experts + n_experts // 8 + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        self.ids[n // 2:n // 2 + 3] = -1
        self.starts, self.rows, self.slots = (torch.full((k + 1,), 77, dtype=torch.int32, device="cuda")
                                              for k in (n_experts + 1, n, n))

    def run(self, ctx):
        ctx.expert_plan_async(self.ids.data_ptr(), self.npos, self.topk, self.n_experts, self.starts.data_ptr(),
                              self.rows.data_ptr(), self.slots.data_ptr())


@pytest.mark.parametrize("npos,topk,n_experts", [(1 << 20, 1, 256), ((1 << 20) - 4096, 1, 300), (1050001, 1, 1), (700001, 3, 5),
                                                 (1000003, 5, 1023), (3000000, 2, 1024), (2500000, 8, 17)])
def test_plans_of_many_routes(ctx, npos, topk, n_experts):
    """From 256 chunks of 4096 routes on, the chunks' counts are added up by a launch of its own."""
    r = Routes(npos, topk, n_experts)
    for _ in range(2):
        r.run(ctx)
    ctx.synchronize()
    n = npos * topk
    key = torch.where((r.ids >= 0) & (r.ids < n_experts), r.ids, n_experts).long()
    order = torch.argsort(key, stable=True)
    starts = torch.cat([key.new_zeros(1), torch.bincount(key, minlength=n_experts + 1)[:n_experts].cumsum(0)])
    listed = int(starts[-1])
    slots = torch.full_like(key, -1)
    slots[order[:listed]] = torch.arange(listed, device="cuda")
    rows = torch.full_like(key, -1)
    rows[:listed] = order[:listed] // topk
    assert torch.equal(r.starts[:-1].long(), starts)
    assert torch.equal(r.rows[:-1].long(), rows) and torch.equal(r.slots[:-1].long(), slots)
    assert r.starts[-1] == r.rows[-1] == r.slots[-1] == 77


def test_a_plan_costs_what_its_routes_do(ctx):
    """Eight times the routes: about eight times as long, where every chunk that adds up
    all others' counts takes 64 times."""
    took = []
    for npos in (1 << 20, 1 << 23):
        r = Routes(npos, 8, 1024)
        r.run(ctx)
        ctx.synchronize()
        best = 1e9
        for _ in range(5):
            torch.cuda.synchronize()
            t = time.perf_counter()
            r.run(ctx)
            ctx.raw.synchronize()
            best = min(best, time.perf_counter() - t)
        took.append(best)
    assert took[1] <= 24 * took[0]


def test_plans_of_one_launch_need_no_call_before_a_capture():
    """Up to 4096 routes a plan uses no memory of the context: the first call of a new one
    is captured."""
    for npos, topk, n_experts in ((4096, 1, 1024), (512, 8, 256), (682, 6, 64)):
        r = Routes(npos, topk, n_experts)
        torch.cuda.synchronize()
        fresh = wa.Context(0)
        g = fresh.graph_capture(lambda: r.run(fresh))
        for _ in range(3):
            r.slots.fill_(77)
            torch.cuda.synchronize()
            fresh.graph_launch(g)
            fresh.synchronize()
            ids = r.ids.cpu().numpy()
            order = np.argsort(np.where((ids >= 0) & (ids < n_experts), ids, n_experts), kind="stable")
            listed = int(r.starts[n_experts])
            want = np.full(npos * topk, -1)
            want[order[:listed]] = np.arange(listed)
            assert listed == ((ids >= 0) & (ids < n_experts)).sum() and np.array_equal(r.slots[:-1].cpu().numpy(), want)
        fresh.graph_release(g)
        fresh.close()


def test_the_widest_tensors(ctx):
    """40704 columns are the most that the resident layout and its products take."""
    rng = np.random.default_rng(1)
    w, s = rng.integers(0, 127, (16, 40832), dtype=np.uint8), np.full((1, 319), 120, np.uint8)
    wide = ctx.store_fp8(w, 16, 40832, s, 1, 319)
    x = Rows(2, 40832)
    y = torch.zeros(2, 16, device="cuda")
    d, sd = torch.from_numpy(w[:, :40704].copy()).cuda(), torch.from_numpy(s[:, :318].copy()).cuda()
    torch.cuda.synchronize()
    with pytest.raises(wa.DeepSeekV4KernelError) as e:
        ctx.fp8_rows_mm_async(wide, 0, 16, x.c, 2, y.data_ptr(), 16, False)
    assert e.value.code == 15
    with pytest.raises(wa.DeepSeekV4KernelError) as e:
        ctx.store_fp8_device(d.data_ptr(), 16, 40832, sd.data_ptr(), 1, 319)  # refused before it is read
    assert e.value.code == 15
    ctx.release(wide)
    h = ctx.store_fp8_device(d.data_ptr(), 16, 40704, sd.data_ptr(), 1, 318)
    x.codes.fill_(0x38)  # 1.0
    x.scales.fill_(127)
    ctx.fp8_rows_mm_async(h, 0, 16, x.c, 2, y.data_ptr(), 16, False)
    ctx.synchronize()
    want = E4M3[w[:, :40704]].sum(1) * 2.0 ** -7
    assert (np.abs(y.cpu().double().numpy() - want) <= 40712 * 2.0 ** -24 * want).all()
    ctx.release(h)


@pytest.mark.parametrize("kind,n", [(THIN, 3), (THIN, 30), (TILE, 300)])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("zero", ["byte 0", 0.0, -0.0])
def test_scales_of_zero_meet_rows_near_the_largest_f32(ctx, kind, n, bf16, zero):
    """x of 448 * 2^120 in a block whose weight scale is 0.0: nothing is added, though the
    block's codes times the row's scale alone are past f32."""
    rows, cols, f32 = 256, 640, zero != "byte 0"
    assert plan(n, rows, cols, f32=f32, bf16=bf16)[0] == kind
    codes = np.full((rows, cols), 0x7E, np.uint8)  # 448
    scales = np.full((2, 5), 2.0 ** -110, np.float32) if f32 else np.full((2, 5), 17, np.uint8)
    scales[0, 1] = scales[1, 0] = zero if f32 else 0
    h = ctx.store_fp8(codes, rows, cols, scales, 2, 5, int(f32))
    r = Rows(n, cols)
    r.codes.fill_(0x7E)
    r.scales.fill_(247)
    y = torch.empty(n, rows, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    ctx.fp8_rows_mm_async(h, 0, rows, r.c, n, y.data_ptr(), rows, bf16)
    ctx.synchronize()
    want = 448.0 * 448 * 128 * 4 * 2.0 ** 10  # four blocks of equal products
    assert bool(((y.double() - want).abs() <= (2.0 ** -8 if bf16 else 648 * 2.0 ** -24) * want).all())
    ctx.release(h)


@pytest.mark.parametrize("kind,n", [(THIN, 3), (THIN, 30), (TILE, 300)])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_infinite_scales_meet_the_smallest_rows(ctx, kind, n, bf16, f32):
    """Rows of 2^-9 * 2^-126, the least that are not 0: infinite with the sign of the product."""
    rows, cols = 256, 640
    assert plan(n, rows, cols, f32=f32, bf16=bf16)[0] == kind
    codes = np.full((rows, cols), 0x01, np.uint8)  # 2^-9
    codes[::2] = 0x81
    scales = np.full((2, 5), 2.0 ** -20, np.float32) if f32 else np.full((2, 5), 107, np.uint8)
    scales[0, 1] = scales[1, 0] = np.inf if f32 else 255
    h = ctx.store_fp8(codes, rows, cols, scales, 2, 5, int(f32))
    r = Rows(n, cols)
    r.codes.fill_(0x01)
    r.scales.fill_(1)
    y = torch.empty(n, rows, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    ctx.fp8_rows_mm_async(h, 0, rows, r.c, n, y.data_ptr(), rows, bf16)
    ctx.synchronize()
    assert bool((y[:, 1::2] == float("inf")).all()) and bool((y[:, ::2] == -float("inf")).all())
    ctx.release(h)
