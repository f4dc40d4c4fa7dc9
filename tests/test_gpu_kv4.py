"""The paged 4-bit attention cache on the GPU: plans, rows in and out and
attention against plain computations in 64 bits, at the sizes and masks where
they can go wrong.

Tolerances are sums of half-step roundings, u = 2^-24 for f32:
  a score of d products added in f32, its query in two f16 parts (2^-22) and
  three factors: (d + 12) u of scale * sum |q||k|, and d u of the largest
  |q| * |k| for what f16 drops 2^-24 below a row's largest; bf16 queries are
  two E4M3 parts of 32 values each, the largest in [2^7, 2^8) and the second
  part in steps of 2^-13 at least: half a step is 2^-21 = 8 u of the largest;
  a weight: twice the largest score error, 4 u of the largest score, and the
  rounding of the weight itself (f32 2^-22, bf16 one f16: 2^-11);
  sums of n weights and products: 2 n + 16 u, and f16's smallest step under
  the largest weight: 2 n u of the largest |v|; bf16 also takes value rows
  against the largest of all, in f16 steps of 2^-24 of at most 16 times the
  largest |v|: 8 u of it;
  the output: 4 u, or half a step of bf16, 2^-8."""
import math

import numpy as np
import pytest
import torch

import wohper_amd as wa

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NONE = 0xFFFFFFFF
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def i32(v):
    return torch.tensor(np.asarray(v, np.int64).astype(np.uint32).view(np.int32), device="cuda")


def u32(t):
    return t.cpu().numpy().view(np.uint32).astype(np.int64)


def ptr(t):
    return t.data_ptr() if t is not None else None


def done(ctx):
    ctx.synchronize()


class Cache:
    """Planes of random bytes (the old contents of reused pages)."""

    def __init__(self, n_pages, page, kv_heads, d, latent, seed=0, codes=None):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.n_pages, self.page, self.kv_heads, self.d, self.latent = n_pages, page, kv_heads, d, latent
        shape = (n_pages, kv_heads, page)

        def old(w):
            return torch.randint(0, 256, (*shape, w), generator=g, device="cuda", dtype=torch.uint8)

        self.planes = [(old(d // 2), old(d // 32)) for _ in range(1 if latent else 2)]
        p = [ptr(t) for pl in self.planes for t in pl] + [None, None]
        self.c = wa.WhKv4Cache(*p[:4], n_pages, page, kv_heads, d)

    def fill(self, plane, slots, rows):
        """Rows [n, kv_heads * d] rounded on the host into the slots."""
        codes, scales = round_rows(rows.reshape(-1, self.kv_heads, self.d))
        page, row = torch.as_tensor(slots // self.page), torch.as_tensor(slots % self.page)
        c, s = self.planes[plane]
        c[page.cuda(), :, row.cuda()] = torch.from_numpy(codes).cuda()
        s[page.cuda(), :, row.cuda()] = torch.from_numpy(scales).cuda()

    def rows(self, plane, slots):
        """f64 [n, kv_heads, d] that the slots stand for."""
        c, s = self.planes[plane]
        page, row = torch.as_tensor(slots // self.page).cuda(), torch.as_tensor(slots % self.page).cuda()
        c, s = c[page, :, row].cpu().numpy(), s[page, :, row].cpu().numpy().astype(int)
        nib = np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], self.d)
        v = GRID[nib & 7] * np.where(nib & 8, -1.0, 1.0)
        scale = np.where(s == 0, 0.0, np.where(s == 255, np.nan, np.exp2(s - 127.0)))
        return v * np.repeat(scale, 32, -1)


def round_rows(x):
    """Codes [.., d / 2] and scale bytes [.., d / 32] of f64 rows, by distance."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], -1, 32)
    top = np.abs(g).max(-1)
    bad = ~np.isfinite(top)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.ceil(np.log2(np.where(bad | (top == 0), 1.0, top) / 6.0))
    e = np.where(top > 6 * np.exp2(e), e + 1, e)
    e = np.where(top <= 6 * np.exp2(e - 1), e - 1, e)
    e = np.maximum(e, -126)
    t = np.abs(np.where(bad[..., None], 0.0, g)) / np.exp2(e)[..., None]
    dist = np.abs(t[..., None] - GRID)
    dist = np.where(GRID * np.exp2(e)[..., None, None] < 2.0 ** 128, dist, np.inf)  # values are finite f32
    near = dist == dist.min(-1, keepdims=True)
    code = near.argmax(-1)
    tie = near.sum(-1) == 2
    code = np.where(tie & (code % 2 == 1), code + 1, code)
    code = np.where(bad[..., None], 0, code + 8 * (np.signbit(g)))
    byte = np.where(bad, 255, np.where(top == 0, 0, e + 127)).astype(np.uint8)
    code = code.reshape(*x.shape[:-1], -1, 2).astype(np.uint8)
    return code[..., 0] | (code[..., 1] << 4), byte


# ---------------------------------------------------------------- plans

def plain_plan(old, new, tables, page, stack, max_tokens):
    pages = lambda n: -(-n // page)  # noqa: E731
    tables, stack = [list(t) for t in tables], list(stack)
    for b, (o, n) in enumerate(zip(old, new)):
        stack += tables[b][pages(n):pages(o)]
    seen = list(stack)
    starts, slots, positions = [0], [], []
    for b, (o, n) in enumerate(zip(old, new)):
        for i in range(pages(o), pages(n)):
            tables[b][i] = stack.pop()
        for p in range(o, n):
            slots.append(tables[b][p // page] * page + p % page)
            positions.append(p)
        starts.append(len(slots))
    pad = max_tokens - len(slots)
    return dict(tables=tables, seen=seen, count=len(stack), starts=starts, slots=slots + [NONE] * pad,
                positions=positions + [0] * pad)


class Plan:
    def __init__(self, old, new, page, spare=3, extra=5, in_place=False, seed=1, width=None, max_tokens=None):
        rng = np.random.default_rng(seed)
        pages = lambda n: -(-n // page)  # noqa: E731
        held = [pages(n) for n in old]
        self.old, self.new, self.page = list(old), list(new), page
        self.n_pages = sum(max(pages(a), pages(b)) for a, b in zip(old, new)) + spare
        self.width = width or max([max(pages(a), pages(b)) for a, b in zip(old, new)] + [0]) + 2
        order = [int(v) for v in rng.permutation(self.n_pages)]
        self.tables, at = [], 0
        for k in held:
            self.tables.append((order[at:at + k] + [77777] * self.width)[:self.width])
            at += k
        self.stack = order[at:]
        tokens = sum(max(0, b - a) for a, b in zip(old, new))
        self.max_tokens = tokens + extra if max_tokens is None else max_tokens
        n = len(old)
        self.d = dict(old=i32(old or [0]), new=i32(new or [0]), tables=i32(self.tables or [[0]]),
                      free=i32(self.stack + [88888] * (self.n_pages - len(self.stack))), count=i32([len(self.stack)]),
                      starts=i32([9] * (n + 1)), slots=i32([9] * max(1, self.max_tokens)),
                      positions=i32([9] * max(1, self.max_tokens)))
        self.d["free_out"] = self.d["free"] if in_place else i32([99999] * self.n_pages)
        self.d["count_out"] = self.d["count"] if in_place else i32([9])
        p = {k: ptr(t) for k, t in self.d.items()}
        self.s = wa.WhKvPlan(n, p["old"], p["new"], p["tables"], self.width, page, self.n_pages, p["free"], p["count"],
                             p["free_out"], p["count_out"], self.max_tokens, p["starts"], p["slots"], p["positions"])

    def got(self):
        return {k: u32(t).tolist() for k, t in self.d.items()}

    def check(self):
        w = plain_plan(self.old, self.new, self.tables, self.page, self.stack, self.max_tokens)
        g = self.got()
        if self.old:
            assert g["tables"] == w["tables"]
        assert g["starts"] == w["starts"]
        assert g["slots"][:self.max_tokens] == w["slots"] and g["positions"][:self.max_tokens] == w["positions"]
        assert g["count_out"] == [w["count"]]
        assert g["free_out"][:len(w["seen"])] == w["seen"]


PLAN_CASES = {
    "one": ([0], [1], 16), "prompt": ([0], [1000], 64), "decode": ([5, 16, 31, 64], [6, 17, 32, 65], 16),
    "page_of_one": ([3, 0, 2], [5, 4, 0], 1), "ends_and_starts": ([100, 33, 0, 64], [0, 30, 70, 64], 32),
    "all_end": ([7, 8, 9], [0, 0, 0], 4), "nothing": ([7, 0, 9], [7, 0, 9], 4), "no_requests": ([], [], 16),
    "cut_back_in_a_page": ([20, 40], [18, 33], 64), "takes_what_is_given": ([640, 0], [0, 640], 64),
}


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", sorted(PLAN_CASES))
def test_plan(ctx, name, in_place):
    old, new, page = PLAN_CASES[name]
    spare = 0 if name == "takes_what_is_given" else 3
    p = Plan(old, new, page, spare=spare, in_place=in_place)
    if name == "takes_what_is_given":  # only the pages given back are there
        assert len(p.stack) == 10
        p.stack = []
        p.d["count"].zero_()
    torch.cuda.synchronize()
    ctx.kv_plan_async(p.s)
    done(ctx)
    p.check()


@pytest.mark.parametrize("n,page,most", [(64, 64, 4000), (65, 16, 300), (1000, 8, 90), (1025, 16, 40), (4096, 4, 20)])
def test_plan_of_many(ctx, n, page, most):
    """Several requests a thread, several workgroups, in place and not."""
    rng = np.random.default_rng(n)
    old, new = rng.integers(0, most, n).tolist(), rng.integers(0, most, n).tolist()
    for in_place in (False, True):
        p = Plan(old, new, page, in_place=in_place, extra=9000)
        torch.cuda.synchronize()
        ctx.kv_plan_async(p.s)
        done(ctx)
        p.check()


@pytest.mark.parametrize("fault,status", [("pages", 11), ("tokens", 6), ("table", 6), ("count", 11)])
def test_plan_that_does_not_fit(ctx, fault, status):
    old, new = [10, 50, 7], [80, 0, 100]
    p = Plan(old, new, 16, spare=0, width=4 if fault == "table" else None, max_tokens=100 if fault == "tokens" else None)
    if fault == "pages":
        p.d["count"].fill_(4)  # four and the four given back: eight of the ten that it takes
    if fault == "count":
        p.d["count"].fill_(p.n_pages + 1)
    before = p.got()
    torch.cuda.synchronize()
    ctx.kv_plan_async(p.s)
    with pytest.raises(wa.DeepSeekV4KernelError) as e:
        ctx.synchronize()
    assert e.value.code == status
    ctx.synchronize()  # reported once
    g = p.got()
    assert g["tables"] == before["tables"] and g["starts"] == [0] * 4 and g["count_out"] == before["count"]
    assert set(g["slots"]) == {NONE} and set(g["positions"]) == {0}
    n = min(before["count"][0], p.n_pages)
    assert g["free_out"][:n] == before["free"][:n]


def test_plan_with_a_bad_page(ctx):
    p = Plan([3], [40], 16)
    p.d["free"][len(p.stack) - 1] = p.n_pages  # the first that is taken: positions 16 .. 31
    torch.cuda.synchronize()
    ctx.kv_plan_async(p.s)
    with pytest.raises(wa.DeepSeekV4KernelError) as e:
        ctx.synchronize()
    assert e.value.code == 10
    slots = p.got()["slots"]
    assert slots[13:29] == [NONE] * 16 and NONE not in slots[:13] + slots[29:37]


# ------------------------------------------------------------ rows in, out

def special_rows(rng, n, width):
    """Rows whose groups meet every rounding: ties, both ends of the scale's
    range, subnormals, zeros of both signs."""
    x = rng.standard_normal((n, width)) * np.exp2(rng.integers(-3, 4, (n, width // 32)).repeat(32, 1))
    g = x.reshape(n, -1, 32)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4) * np.where(np.arange(32) % 3, 1, -1)
    flat = g.reshape(-1, 32)
    k = len(flat)
    for i, e in enumerate([0, 5, -20, 100, -126, -130]):
        flat[(7 * i) % k] = ties * 2.0 ** e
    flat[(7 * 6 + 1) % k] = 0.0
    flat[(7 * 6 + 2) % k] = -0.0
    flat[(7 * 6 + 3) % k] = 2.0 ** -140 * np.arange(32)
    flat[(7 * 6 + 4) % k] = np.linspace(-3.3e38, 3.3e38, 32)
    flat[(7 * 6 + 5) % k] = np.linspace(0, 6.0000005, 32)
    return x


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("kv_heads,d,page,latent,n", [(1, 512, 64, True, 1), (1, 512, 64, True, 130), (3, 64, 16, False, 33),
                                                      (8, 128, 16, False, 257), (2, 256, 1, False, 9), (1, 64, 8, True, 5)])
def test_rows_in_and_out(ctx, kv_heads, d, page, latent, n, bf16):
    rng = np.random.default_rng(d + n)
    width, n_pages = kv_heads * d, -(-n // page) + 2
    c = Cache(n_pages, page, kv_heads, d, latent)
    before = [(a.clone(), b.clone()) for a, b in c.planes]
    slots = rng.permutation(n_pages * page)[:n]
    passed = np.zeros(n, bool)
    passed[n // 2:n // 2 + 2] = n > 5  # rows of no slot
    given = np.where(passed, NONE, slots)
    stride = width + 24  # rows further apart than they are long
    dt = torch.bfloat16 if bf16 else torch.float32
    rows, ins = [], []
    for k in range(len(c.planes)):
        t = torch.zeros(n, stride, dtype=dt, device="cuda")
        t[:, :width] = torch.from_numpy(special_rows(rng, n, width)).to(dt)
        ins.append(t)
        rows.append(t[:, :width].double().cpu().numpy())
    outs = [torch.full((n, stride), 7.0, dtype=dt, device="cuda") for _ in ins]
    sl = i32(given)
    two = len(ins) == 2
    torch.cuda.synchronize()
    ctx.kv4_write_async(c.c, ptr(ins[0]), stride, ptr(ins[1]) if two else None, stride, bf16, ptr(sl), n)
    ctx.kv4_read_async(c.c, ptr(sl), n, ptr(outs[0]), stride, ptr(outs[1]) if two else None, stride, bf16)
    done(ctx)
    for k, x in enumerate(rows):
        codes, scales = round_rows(x.reshape(n, kv_heads, d))
        want_c, want_s = before[k]
        at = torch.from_numpy(slots[~passed]).cuda()
        want_c[at // page, :, at % page] = torch.from_numpy(codes[~passed]).cuda()
        want_s[at // page, :, at % page] = torch.from_numpy(scales[~passed]).cuda()
        assert torch.equal(c.planes[k][0], want_c) and torch.equal(c.planes[k][1], want_s)
        got = outs[k].double().cpu().numpy()
        assert np.array_equal(got[~passed, :width], c.rows(k, slots[~passed]).reshape(-1, width))
        assert (got[passed] == 7.0).all() and (got[:, width:] == 7.0).all()
    if two:  # either alone
        alone = torch.zeros(n, width, dtype=dt, device="cuda")
        torch.cuda.synchronize()
        ctx.kv4_read_async(c.c, ptr(sl), n, None, 0, ptr(alone), width, bf16)
        done(ctx)
        assert torch.equal(alone[torch.from_numpy(~passed).cuda()], outs[1][torch.from_numpy(~passed).cuda(), :width])


def test_rows_that_are_not_finite(ctx):
    c = Cache(2, 16, 1, 128, True)
    x = torch.randn(3, 128, device="cuda")
    x[0, 5], x[1, 40], x[2, 127] = math.inf, math.nan, -math.inf
    out = torch.zeros_like(x)
    sl = i32([4, 31, 0])
    torch.cuda.synchronize()
    ctx.kv4_write_async(c.c, ptr(x), 128, None, 0, False, ptr(sl), 3)
    ctx.kv4_read_async(c.c, ptr(sl), 3, ptr(out), 128, None, 0, False)
    done(ctx)
    bad = torch.isnan(out).reshape(3, 4, 32)
    want = torch.zeros(3, 4, dtype=torch.bool, device="cuda")
    want[0, 0] = want[1, 1] = want[2, 3] = True
    assert torch.equal(bad.all(-1), want) and torch.equal(bad.any(-1), want)
    assert np.array_equal(out.double().cpu().numpy(), c.rows(0, np.array([4, 31, 0])).reshape(3, -1), equal_nan=True)


def test_slots_behind_the_cache(ctx):
    c = Cache(3, 16, 1, 64, True)
    before = [t.clone() for t in c.planes[0]]
    x = torch.randn(2, 64, device="cuda")
    out = torch.full_like(x, 5.0)
    for slot in (48, 0xFFFFFFFE):
        sl = i32([slot, NONE])
        torch.cuda.synchronize()
        for call in (lambda: ctx.kv4_write_async(c.c, ptr(x), 64, None, 0, False, ptr(sl), 2),
                     lambda: ctx.kv4_read_async(c.c, ptr(sl), 2, ptr(out), 64, None, 0, False)):
            call()
            with pytest.raises(wa.DeepSeekV4KernelError) as e:
                ctx.synchronize()
            assert e.value.code == 10
    assert torch.equal(before[0], c.planes[0][0]) and torch.equal(before[1], c.planes[0][1]) and (out == 5.0).all()


# -------------------------------------------------------------- attention

class Case:
    """Requests with q new tokens of their `lens` cached rows."""

    def __init__(self, q_lens, lens, heads, kv_heads, d, latent, bf16, page=16, window=0, first=0, sink=False, seed=0,
                 pad=0, behind=0, q_scale=2.0, splits_len=None):
        rng = np.random.default_rng(seed + 1000 * d + heads)
        self.__dict__.update(locals())
        counts = [-(-n // page) for n in lens]
        self.n_pages, self.stride = sum(counts) + 2, max(counts + [1]) + 1
        self.cache = Cache(self.n_pages, page, kv_heads, d, latent, seed)
        order = rng.permutation(self.n_pages)
        tables = rng.integers(0, 1 << 32, (len(lens), self.stride))  # past a request's pages: anything
        at, self.slots = 0, []
        for b, n in enumerate(lens):
            tables[b, :counts[b]] = order[at:at + counts[b]]
            at += counts[b]
            pos = np.arange(n)
            s = tables[b][pos // page] * page + pos % page if n else np.zeros(0, int)
            self.slots.append(s)
            for k in range(len(self.cache.planes)):
                x = rng.standard_normal((n, kv_heads * d)) * np.exp2(rng.integers(-2, 3, (n, kv_heads * d // 32)).repeat(32, 1))
                if n:
                    self.cache.fill(k, s, x)
        self.tables = i32(tables)
        self.n_tokens = sum(q_lens) + behind
        self.dt = torch.bfloat16 if bf16 else torch.float32
        width = heads * d
        self.q = torch.zeros(self.n_tokens, width + pad, dtype=self.dt, device="cuda")
        self.q[:, :width] = torch.from_numpy(q_scale * rng.standard_normal((self.n_tokens, width))).to(self.dt)
        self.out = torch.full((self.n_tokens, width + 2 * pad), 7.0, dtype=self.dt, device="cuda")
        self.sinks = torch.from_numpy(rng.standard_normal(heads)).float().cuda() if sink else None
        self.starts = i32(np.concatenate([[0], np.cumsum(q_lens)]))
        self.lens_dev = i32(lens)
        self.scale = float(np.float32(d ** -0.5))

    def desc(self):
        return wa.WhKv4Attention(ptr(self.q), self.q.shape[1], ptr(self.out), self.out.shape[1], int(self.bf16),
                                 self.n_tokens, len(self.lens), ptr(self.starts), ptr(self.lens_dev), ptr(self.tables),
                                 self.stride, self.splits_len or max(self.lens), self.heads, self.scale, self.window,
                                 self.first, ptr(self.sinks))

    def run(self, ctx):
        self.d_ = self.desc()
        torch.cuda.synchronize()
        ctx.kv4_attention_async(self.cache.c, self.d_)
        done(ctx)
        return self.out

    def expect(self):
        """Outputs [n, heads * d] and their tolerance."""
        G, d, at = self.heads // self.kv_heads, self.d, 0
        outs, tols = [], []
        for b, (nq, n) in enumerate(zip(self.q_lens, self.lens)):
            q = self.q[at:at + nq, :self.heads * d].double().reshape(nq, self.heads, d)
            at += nq
            out, tol = torch.zeros_like(q), torch.zeros_like(q)
            pos = n - nq + torch.arange(nq, device="cuda")
            j = torch.arange(n, device="cuda")
            see = j[None] <= pos[:, None]
            if self.window:
                see &= (j[None] > pos[:, None] - self.window) | (j[None] < self.first)
            if n:
                ks = torch.from_numpy(self.cache.rows(0, self.slots[b])).cuda()
                vs = ks if self.latent else torch.from_numpy(self.cache.rows(1, self.slots[b])).cuda()
            for h in range(self.heads):
                if not n:
                    continue
                k, v = ks[:, h // G], vs[:, h // G]
                s = (q[:, h] @ k.T) * self.scale
                s = s.masked_fill(~see, -math.inf)
                sink = self.sinks[h].double() if self.sink else torch.tensor(-math.inf, device="cuda").double()
                top = torch.maximum(s.amax(1), sink)
                w = torch.where(see, torch.exp(s - top.clamp_min(-1e300)[:, None]), 0.0)
                tot = w.sum(1) + (torch.exp(sink - top) if self.sink else 0.0)
                w = torch.where(tot[:, None] > 0, w / tot[:, None], 0.0)
                out[:, h] = w @ v
                W = w @ v.abs()
                big = torch.where(see, s.abs(), 0.0).amax(1)
                ab = torch.where(see, q[:, h].abs() @ k.abs().T, 0.0).amax(1)
                km = torch.where(see, k.abs().amax(1)[None], 0.0).amax(1)
                vm = torch.where(see, v.abs().amax(1)[None], 0.0).amax(1)
                cnt = see.sum(1)
                delta = abs(self.scale) * ((d + 12) * U * ab + (8 if self.bf16 else 1) * d * U * q[:, h].abs().amax(1) * km)
                rel = 2 * delta + 4 * U * big + (2 * cnt + 16) * U + (2.0 ** -11 if self.bf16 else 2.0 ** -22)
                tol[:, h] = rel[:, None] * W + ((2 * cnt + 8) * U * vm)[:, None] + (2.0 ** -8 if self.bf16 else 4 * U) * out[:, h].abs()
            outs.append(out.flatten(1))
            tols.append(tol.flatten(1))
        return torch.cat(outs), torch.cat(tols)

    def check(self, ctx):
        got = self.run(ctx).double()
        want, tol = self.expect()
        n, width = want.shape
        off = (got[:n, :width] - want).abs()
        assert bool((off <= tol).all()), f"{float((off / tol.clamp_min(1e-300)).max()):.3g} of the tolerance"
        assert bool((got[n:] == 7.0).all()) and bool((got[:, width:] == 7.0).all())
        return float((off / tol.clamp_min(1e-300)).max())


LAYOUTS = {  # heads, kv_heads, head_dim, latent
    "latent": (64, 1, 512, True), "latent_50": (50, 1, 512, True), "latent_128": (128, 1, 512, True),
    "latent_16": (16, 1, 512, True), "one": (1, 1, 64, False), "pairs": (6, 3, 64, False), "group_8": (16, 2, 128, False),
    "group_1": (3, 3, 128, False), "group_5": (10, 2, 256, False), "wide": (4, 2, 512, False), "group_20": (40, 2, 128, False),
    "latent_64": (8, 1, 64, True), "latent_256": (20, 1, 256, True), "group_40": (80, 2, 64, False),
}
LENGTHS = {  # new tokens and cached rows of each request, page
    "one_of_one": ([1], [1], 16), "decode": ([1, 1, 1], [33, 100, 64], 16), "verify": ([4, 2, 5], [40, 7, 5], 8),
    "prompt": ([70, 1, 17], [70, 90, 33], 16), "page_of_one": ([2, 3], [9, 20], 1), "uneven": ([3, 0, 1], [31, 65, 129], 64),
}


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("layout", sorted(LAYOUTS))
def test_attention(ctx, layout, lengths, bf16):
    q, lens, page = LENGTHS[lengths]
    Case(q, lens, *LAYOUTS[layout], bf16, page=page, sink=len(layout) % 2 == 0).check(ctx)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("window,first", [(1, 0), (1, 3), (16, 0), (17, 4), (40, 1), (64, 64), (1000, 7), (1 << 40, 5)])
@pytest.mark.parametrize("layout", ["latent", "pairs", "group_8"])
def test_windows_and_first_tokens(ctx, layout, window, first, bf16):
    Case([1, 6, 75], [90, 200, 130], *LAYOUTS[layout], bf16, window=window, first=first, seed=window % 97).check(ctx)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout,q,lens", [("latent", [1], [4097]), ("latent", [1, 2], [3000, 500]), ("group_8", [1], [9001]),
                                           ("group_8", [1, 1, 3], [5000, 31, 2050]), ("pairs", [1], [6000]),
                                           ("latent_256", [2], [2500])])
def test_long_keys_are_split_and_joined(ctx, layout, q, lens, bf16):
    Case(q, lens, *LAYOUTS[layout], bf16, page=64, sink=True).check(ctx)


@pytest.mark.parametrize("window,first", [(0, 0), (700, 5)])
@pytest.mark.parametrize("layout", ["latent", "group_8", "group_5", "latent_50"])
def test_equal_weights_are_exact(ctx, layout, window, first):
    """Queries of zero: weights are one power of two, sums of small multiples
    of powers of two are exact, so a key too many or too few shows at any
    length; the divisions and the join round (splits + 8 times)."""
    c = Case([1, 40], [5000, 1500], *LAYOUTS[layout], False, page=64, window=window, first=first, q_scale=0.0)
    got = c.run(ctx).double()
    want, _ = c.expect()
    tops = []
    for b, n in enumerate(c.lens):
        v = np.abs(c.cache.rows(len(c.cache.planes) - 1, c.slots[b])).max()
        tops.append(v)
    assert bool(((got - want).abs() <= (64 + 8) * U * max(tops)).all())


def test_one_visible_key_is_returned_as_it_is(ctx):
    """A weight of one: f32 outputs are the cached values."""
    for layout in ("latent", "pairs", "group_8"):
        c = Case([1], [200], *LAYOUTS[layout], False, window=1)
        got = c.run(ctx).double().cpu().numpy()
        v = c.cache.rows(len(c.cache.planes) - 1, c.slots[0][-1:])[0]
        want = np.repeat(v, c.heads // c.kv_heads, 0).reshape(1, -1)
        assert np.abs(got - want).max() <= 2 * U * np.abs(want).max()


@pytest.mark.parametrize("sink", [False, True])
def test_rows_that_see_nothing_are_zero(ctx, sink):
    """Requests of no rows, and more tokens than rows: the first see nothing."""
    c = Case([2, 4, 1], [0, 2, 5], *LAYOUTS["group_8"], False, sink=sink)
    got = c.run(ctx)
    assert bool((got[:4] == 0).all()) and bool((got[4:] != 0).any(1).all())
    want, tol = c.expect()
    assert bool(((got.double() - want).abs() <= tol).all())


def test_rows_behind_the_last_request_stay(ctx):
    c = Case([3, 20], [30, 40], *LAYOUTS["pairs"], False, behind=37, pad=8)
    c.check(ctx)


@pytest.mark.parametrize("bf16", [False, True])
def test_strides(ctx, bf16):
    Case([2, 19], [50, 19], *LAYOUTS["group_5"], bf16, pad=8).check(ctx)


@pytest.mark.parametrize("layout", ["latent", "group_8", "pairs"])
def test_keys_that_are_not_finite(ctx, layout):
    """NaN in a row that nobody sees does nothing; in one that some tokens see
    it reaches those tokens and the heads of that key head only."""
    for where, plane in ((0, 0), (0, -1), (39, 0), (39, -1)):
        c = Case([6], [40], *LAYOUTS[layout], False, window=20)
        ref = c.run(ctx).clone()
        slot = int(c.slots[0][where])
        c.cache.planes[plane][1][slot // c.page, 0, slot % c.page, 1] = 255
        c.out.fill_(7.0)
        got = c.run(ctx)
        if where == 0:  # outside every window
            assert torch.equal(got, ref)
        else:  # the last token's own row, of key head 0
            assert torch.equal(got[:5], ref[:5])
            g = c.heads // c.kv_heads
            last = got[5].reshape(c.heads, c.d)
            assert bool(torch.isnan(last[:g]).all()) and torch.equal(last[g:], ref[5].reshape(c.heads, c.d)[g:])


def test_scales_far_apart(ctx):
    """Rows and groups from 2^-60 to 2^60 of each other, both ends first."""
    for latent, d in ((True, 512), (False, 128)):
        c = Case([2], [96], 4, 1, d, latent, False, q_scale=1.0)
        rng = np.random.default_rng(5)
        e = np.concatenate([np.linspace(-60, 0, 48), np.linspace(60, -60, 48)])
        if latent:
            e = np.minimum(e, 0)  # scores stay finite in the exponential
        for k in range(len(c.cache.planes)):
            x = rng.standard_normal((96, d))
            if k or latent:
                x = x * np.exp2(np.round(e))[:, None] * np.exp2(rng.integers(-12, 1, (96, d // 32)).repeat(32, 1))
            c.cache.fill(k, c.slots[0], x)
        c.check(ctx)


def test_all_zero_rows(ctx):
    c = Case([3], [50], *LAYOUTS["latent"], False, sink=True)
    c.cache.fill(0, c.slots[0], np.zeros((50, 512)))
    assert bool((c.run(ctx) == 0).all())


def test_large_scores(ctx):
    """A score far above the others, arriving last and first."""
    for at in (0, 170, 199):
        c = Case([1], [200], *LAYOUTS["group_8"], False, q_scale=8.0)
        k = c.cache.rows(0, c.slots[0]).reshape(200, -1)
        k[at] *= 8
        c.cache.fill(0, c.slots[0], k)
        c.check(ctx)


def test_bad_pages_and_lengths_are_reported(ctx):
    for what in ("page", "length"):
        c = Case([2], [40], *LAYOUTS["group_8"], False)
        if what == "page":
            c.tables[0, 1] = c.n_pages
        else:
            c.lens_dev[0] = 16 * c.stride + 1
            c.tables.fill_(0)
        d = c.desc()
        torch.cuda.synchronize()
        ctx.kv4_attention_async(c.cache.c, d)
        with pytest.raises(wa.DeepSeekV4KernelError) as e:
            ctx.synchronize()
        assert e.value.code == 10
        ctx.synchronize()


def test_offsets_past_32_bits(ctx):
    """A cache of 4.6 GB of codes whose request lies on its last pages."""
    n_pages, page = 18 << 14, 64
    free = torch.cuda.mem_get_info()[0]
    assert free > 8 << 30
    c = Case([2], [300], *LAYOUTS["latent"], True, page=page)
    codes = torch.zeros(n_pages, 1, page, 256, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(n_pages, 1, page, 16, dtype=torch.uint8, device="cuda")
    small = c.cache
    k = -(-300 // page)
    tables = u32(c.tables)[0]
    for i in range(k):
        codes[n_pages - 1 - i], scales[n_pages - 1 - i] = small.planes[0][0][tables[i]], small.planes[0][1][tables[i]]
    want, tol = c.expect()
    c.tables[0, :k] = torch.arange(n_pages - 1, n_pages - 1 - k, -1, device="cuda").int()
    c.cache = type("C", (), dict(c=wa.WhKv4Cache(ptr(codes), ptr(scales), None, None, n_pages, page, 1, 512)))()
    got = c.run(ctx).double()
    assert bool(((got - want).abs() <= tol).all())
    out = torch.zeros(300, 512, device="cuda")
    pos = torch.arange(300, device="cuda")
    sl = (c.tables[0][pos // page] * page + pos % page).int()
    torch.cuda.synchronize()
    ctx.kv4_read_async(c.cache.c, ptr(sl), 300, ptr(out), 512, None, 0, False)
    done(ctx)
    assert np.array_equal(out.double().cpu().numpy(), small.rows(0, c.slots[0]).reshape(300, -1))


def test_results_repeat_bit_for_bit(ctx):
    for layout, q, lens in (("latent", [1, 1], [3000, 700]), ("group_8", [9, 1], [9, 4000])):
        c = Case(q, lens, *LAYOUTS[layout], False, page=64)
        first = c.run(ctx).clone()
        for _ in range(5):
            c.out.fill_(7.0)
            assert torch.equal(c.run(ctx), first)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout,q", [("latent", [1]), ("latent", [40]), ("group_8", [3]), ("group_8", [90]), ("latent_64", [50])])
def test_keys_that_are_not_finite_in_long_lists(ctx, layout, q, bf16):
    """The same past the first run of keys, in both kinds of tile: NaN reaches
    the tokens whose window holds the key and no others."""
    n, window = 400, 100
    for key in (150, 310, 396):
        for plane in (0, -1):
            c = Case(q, [n], *LAYOUTS[layout], bf16, window=window, page=64)
            ref = c.run(ctx).clone()
            slot = int(c.slots[0][key])
            c.cache.planes[plane][1][slot // c.page, 0, slot % c.page, -1] = 255
            c.out.fill_(7.0)
            got = c.run(ctx)
            pos = n - q[0] + torch.arange(q[0], device="cuda")
            sees = (pos >= key) & (pos - window < key)
            g = c.heads // c.kv_heads
            nan = torch.isnan(got.reshape(q[0], c.heads, c.d))
            assert bool(nan[sees, :g].all()) and not bool(nan[~sees].any()) and not bool(nan[:, g:].any())
            assert torch.equal(got[~sees], ref[~sees])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout,q", [("group_8", [1]), ("group_8", [60]), ("pairs", [2]), ("group_5", [30]), ("wide", [1]), ("group_40", [4])])
def test_value_scales_that_rise(ctx, layout, q, bf16):
    """Values that grow with the key by 2^40 over the list, so that what was
    added up is taken against a new reference many times."""
    c = Case(q, [500], *LAYOUTS[layout], bf16, page=64, sink=True)
    rng = np.random.default_rng(3)
    x = rng.standard_normal((500, c.kv_heads * c.d)) * np.exp2(np.arange(500) * 40 // 500 - 20.0)[:, None]
    c.cache.fill(1, c.slots[0], x)
    c.check(ctx)


@pytest.mark.parametrize("requests", [70, 200, 300])
def test_many_requests_with_none_between(ctx, requests):
    """Lengths from 0 to some thousands, tokens from none to three, over and
    under the number of requests that a split counts."""
    rng = np.random.default_rng(requests)
    q = [int(v) for v in rng.integers(0, 4, requests)]
    q[0], q[-1] = 0, 0
    lens = [max(n, int(v)) for n, v in zip(q, np.exp2(rng.uniform(0, 9, requests)))]
    lens[requests // 2] = 4000
    q[requests // 2] = 2
    for layout in ("group_8", "latent_64"):
        Case(q, lens, *LAYOUTS[layout], True, page=32, behind=3).check(ctx)


@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30])
@pytest.mark.parametrize("layout,q", [("latent", [2]), ("group_8", [1]), ("group_8", [70])])
def test_other_scales(ctx, layout, q, scale):
    for bf16 in (False, True):
        c = Case(q, [200], *LAYOUTS[layout], bf16, window=150, first=3, sink=True)
        c.scale = float(np.float32(scale))
        c.check(ctx)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout,q,lens,window,first", [
    ("group_8", [1], [6000], 3000, 0), ("group_8", [3, 1], [6000, 100], 2500, 130), ("latent", [1], [3000], 1000, 64),
    ("latent", [2], [3000], 1500, 7), ("latent_16", [1, 1], [5000, 64], 4095, 1)])
def test_windows_of_split_lists(ctx, layout, q, lens, window, first, bf16):
    Case(q, lens, *LAYOUTS[layout], bf16, page=64, window=window, first=first).check(ctx)


@pytest.mark.parametrize("page", [8, 64, 256])
@pytest.mark.parametrize("layout,q", [("group_8", [1]), ("group_8", [70]), ("latent", [1, 3]), ("latent", [1])])
@pytest.mark.parametrize("window,first", [(100, 0), (100, 5), (300, 70), (65, 64)])
def test_pages_that_no_token_sees_need_no_entry(ctx, layout, q, page, window, first):
    lens = [1111, 700][:len(q)]
    c = Case(q, lens, *LAYOUTS[layout], False, page=page, window=window, first=first)
    tables = u32(c.tables).reshape(len(q), -1)
    for b, (nq, n) in enumerate(zip(q, lens)):
        seen = np.zeros(n, bool)
        seen[:first] = True
        seen[max(0, n - nq + 1 - window):] = True
        for p in range(-(-n // page)):
            if not seen[p * page:(p + 1) * page].any():
                tables[b, p] = 0xFFFFFFFF - p
    c.tables = i32(tables)
    c.check(ctx)


def test_graphs_that_share_scratch(ctx):
    """Two captured calls whose key lists are split use the same scratch: in
    any order, with an eager one between, each gives its own result."""
    cases = [Case([1], [5000], *LAYOUTS["group_8"], True, page=64), Case([1, 1], [3000, 900], *LAYOUTS["latent"], False, page=16),
             Case([2], [2500], *LAYOUTS["group_5"], False, page=64)]
    want = [c.run(ctx).clone() for c in cases]
    graphs = [ctx.graph_capture(lambda c=c: ctx.kv4_attention_async(c.cache.c, c.d_)) for c in cases[:2]]
    for order in ((0, 1), (1, 0), (0, 0), (1, 1)):
        for c in cases:
            c.out.fill_(7.0)
        torch.cuda.synchronize()
        for k in order:
            ctx.graph_launch(graphs[k])
        ctx.kv4_attention_async(cases[2].cache.c, cases[2].d_)
        done(ctx)
        assert torch.equal(cases[2].out, want[2])
        for k in set(order):
            assert torch.equal(cases[k].out, want[k])
    for g in graphs:
        ctx.graph_release(g)


def test_two_contexts_at_once():
    """Each context has its own stream and scratch."""
    with wa.Context(0) as one, wa.Context(0) as two:
        cases = [Case([1], [5000], *LAYOUTS["group_8"], True, page=64), Case([1], [4000], *LAYOUTS["latent"], True, page=64)]
        want = [c.run(one).clone() for c in cases]
        for _ in range(4):
            for c in cases:
                c.out.fill_(7.0)
            torch.cuda.synchronize()
            for c, k in zip(cases, (one, two)):
                k.kv4_attention_async(c.cache.c, c.d_)
            done(one)
            done(two)
            assert all(torch.equal(c.out, w) for c, w in zip(cases, want))


# ------------------------------------------------------- the calls together

def serving_step(ctx, heads, kv_heads, d, latent, bf16, steps=6):
    """A decode loop of its own lengths: plan in place, rows in, attention;
    yields each step's results and what they should be."""
    rng = np.random.default_rng(d)
    page, n = 8, 4
    lens = [0, 0, 0, 0]
    cache = Cache(64, page, kv_heads, d, latent)
    tables = torch.zeros(n, 12, dtype=torch.int32, device="cuda")
    free, count = i32(rng.permutation(64)), i32([64])
    dt = torch.bfloat16 if bf16 else torch.float32
    width, T = heads * d, 48
    bufs = dict(old=i32(lens), new=i32(lens), starts=i32([0] * (n + 1)), slots=i32([0] * T), pos=i32([0] * T),
                q=torch.zeros(T, width, dtype=dt, device="cuda"), out=torch.zeros(T, width, dtype=dt, device="cuda"),
                k=torch.zeros(T, kv_heads * d, dtype=dt, device="cuda"), v=torch.zeros(T, kv_heads * d, dtype=dt, device="cuda"))
    bufs.update(tables=tables, free=free, count=count)  # kept as long as the descriptors below
    plan = wa.WhKvPlan(n, ptr(bufs["old"]), ptr(bufs["new"]), ptr(tables), 12, page, 64, ptr(free), ptr(count), ptr(free),
                       ptr(count), T, ptr(bufs["starts"]), ptr(bufs["slots"]), ptr(bufs["pos"]))
    att = wa.WhKv4Attention(ptr(bufs["q"]), width, ptr(bufs["out"]), width, int(bf16), T, n, ptr(bufs["starts"]),
                            ptr(bufs["new"]), ptr(tables), 12, 96, heads, d ** -0.5, 0, 0, None)

    def step():
        ctx.kv_plan_async(plan)
        ctx.kv4_write_async(cache.c, ptr(bufs["k"]), kv_heads * d, None if latent else ptr(bufs["v"]), kv_heads * d, bf16,
                            ptr(bufs["slots"]), T)
        ctx.kv4_attention_async(cache.c, att)

    history = [[np.zeros((0, kv_heads, d)) for _ in range(n)] for _ in range(2)]
    targets = [[20, 3, 0, 9], [21, 4, 17, 9], [22, 2, 18, 10], [0, 5, 19, 40], [8, 6, 20, 41], [9, 7, 21, 42]][:steps]

    def feed(i):
        new = targets[i]
        bufs["old"].copy_(i32(lens))
        bufs["new"].copy_(i32(new))
        for k in ("q", "k", "v"):
            bufs[k].copy_(torch.from_numpy(rng.standard_normal(tuple(bufs[k].shape))).to(dt))
        bufs["out"].fill_(7.0)
        torch.cuda.synchronize()

    def check(i):
        new, at = targets[i], 0
        got = bufs["out"].double().cpu().numpy()
        for b in range(n):
            for p, name in enumerate(("k", "v")):
                rows = bufs[name].double().cpu().numpy().reshape(T, kv_heads, d)
                codes, scales = round_rows(rows)
                nib = np.stack([codes & 15, codes >> 4], -1).reshape(rows.shape)
                val = GRID[nib & 7] * np.where(nib & 8, -1.0, 1.0) * np.repeat(np.exp2(scales.astype(int) - 127.0), 32, -1)
                grown = max(0, new[b] - lens[b])
                history[p][b] = np.concatenate([history[p][b][:new[b]], val[at:at + grown]])
            grown = max(0, new[b] - lens[b])
            assert len(history[0][b]) == new[b]
            ks, vs = history[0][b], history[0][b] if latent else history[1][b]
            for t in range(grown):
                for h in range(heads):
                    q = bufs["q"][at + t].double().cpu().numpy().reshape(heads, d)[h]
                    m = new[b] - grown + t + 1
                    s = ks[:m, h // (heads // kv_heads)] @ q * d ** -0.5
                    w = np.exp(s - s.max())
                    want = w / w.sum() @ vs[:m, h // (heads // kv_heads)]
                    off = np.abs(got[at + t].reshape(heads, d)[h] - want).max()
                    # scores of order 3 and values up to 12: twice 600 u of sum |q||k|, and half a step of bf16
                    assert off <= (2.0 ** -7 if bf16 else 2.0 ** -12) * np.abs(vs[:m]).max()
            at += grown
        assert (got[at:] == 7.0).all()
        lens[:] = new

    return step, feed, check, len(targets), bufs


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv_heads,d,latent", [(20, 1, 512, True), (8, 2, 128, False)])
def test_a_decode_loop(ctx, heads, kv_heads, d, latent, bf16):
    step, feed, check, n, _ = serving_step(ctx, heads, kv_heads, d, latent, bf16)
    for i in range(n):
        feed(i)
        step()
        done(ctx)
        check(i)


def test_a_captured_step_follows_its_lengths(ctx):
    """One graph for every step: lengths, slots and results are the replay's
    own, with eager calls of the same operators between."""
    step, feed, check, n, _ = serving_step(ctx, 8, 2, 128, False, False)
    other = Case([1, 3], [500, 40], *LAYOUTS["latent"], False)
    ref = other.run(ctx).clone()
    # sizes the context's scratch without moving the loop's state: old and new lengths are 0 here
    step()
    done(ctx)
    graph = ctx.graph_capture(step)
    for i in range(n):
        feed(i)
        ctx.graph_launch(graph)
        done(ctx)
        check(i)
        other.out.fill_(7.0)
        assert torch.equal(other.run(ctx), ref)
    ctx.graph_release(graph)
