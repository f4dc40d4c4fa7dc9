"""4-bit cache attention over values, keys and queries whose sizes lie far apart.

An output is a sum over the keys that its row sees: neither a row that only a
later token sees, nor a row of no weight, nor another group of 32 dims may cost
it bits.  So the tolerance has no term of the largest |v|:

  u = 2^-24.  |error| <= (2 delta + 4 u S + (2 n + 16) u + r) sum w g + o |out|
  g: the largest |v| of the value's own group of 32 dims
  delta: a score's error, (d + 12) u scale sum |q||k| for d f32 products, the
    query's two f16 parts and three factors (the second part ends 2^-48 below the
    query's largest value, 2^-25 where keys are 2^23 the other way); bf16 queries (two E4M3 parts of 32
    values) add 8 u of the largest |q| times the largest |k| for each of a group's dims
  S: the largest score, whose rounding in the exponent the weights carry; where
    the weight's reference includes a value's exponent, at most 40 and 6 more of
    such powers of two: 48 u
  (2 n + 16) u: sums of n weights and n products, n u of each; and what two
    halves of f16 leave below their last bit: with weights times 2^8 under a
    reference R = max w 2^(row's exponent), half a step of 2^-24 is 2^-33 R, for
    n terms.  A group lies at most 2^9 below its row there, so R is at most 2^9
    times the largest w 2^(group's exponent), which is at most w g / 3: n terms of
    2^-33 2^9 / 3 = u / 3 of max w g (bf16 2^12: 3 u, of n = 130 terms 2^-15.4, a
    twentieth of r)
  r: a weight's own rounding, 2^-22 (two f16 parts) or 2^-11 (bf16: one)
  o: the output's, 4 u, or half a step of bf16, 2^-8
The sums here are short, so that the term of n stays below 2^-15."""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv4 import LAYOUTS, U, Case, ptr

pytestmark = pytest.mark.gpu


def bound(c, tiny=0.0):
    """Outputs [n, heads * d] in 64 bits and their tolerance; tiny: an absolute
    term for outputs at the lower end of f32."""
    G, d, at = c.heads // c.kv_heads, c.d, 0
    outs, tols = [], []
    for b, (nq, n) in enumerate(zip(c.q_lens, c.lens)):
        q = c.q[at:at + nq, :c.heads * d].double().reshape(nq, c.heads, d)
        at += nq
        out, tol = torch.zeros_like(q), torch.zeros_like(q)
        pos, j = n - nq + torch.arange(nq, device="cuda"), torch.arange(n, device="cuda")
        see = j[None] <= pos[:, None]
        if c.window:
            see &= (j[None] > pos[:, None] - c.window) | (j[None] < c.first)
        ks = torch.from_numpy(c.cache.rows(0, c.slots[b])).cuda()
        vs = ks if c.latent else torch.from_numpy(c.cache.rows(1, c.slots[b])).cuda()
        for h in range(c.heads):
            k, v = ks[:, h // G], vs[:, h // G]
            s = torch.where(see, (q[:, h] @ k.T) * c.scale, -math.inf)
            sink = c.sinks[h].double() if c.sink else torch.tensor(-math.inf, device="cuda").double()
            top = torch.maximum(s.amax(1), sink)
            w = torch.exp(s - top[:, None])
            w = w / (w.sum(1) + torch.exp(sink - top))[:, None]
            ab = torch.where(see, q[:, h].abs() @ k.abs().T, 0.0).amax(1)
            qg, kg = q[:, h].abs().reshape(nq, -1, 32).amax(2), k.abs().reshape(n, -1, 32).amax(2)
            by_group = torch.where(see, 32 * (qg @ kg.T), 0.0).amax(1)
            delta = abs(c.scale) * ((d + 12) * U * ab + (8 * U * by_group if c.bf16 else 0.0))
            big = torch.where(see, s.abs(), 0.0).amax(1)
            rel = 2 * delta + 4 * U * big + 48 * U + (2 * see.sum(1) + 16) * U + (2.0 ** -11 if c.bf16 else 2.0 ** -22)
            out[:, h] = w @ v
            g = v.abs().reshape(n, -1, 32).amax(2).repeat_interleave(32, 1)
            tol[:, h] = rel[:, None] * (w @ g) + (2.0 ** -8 if c.bf16 else 4 * U) * out[:, h].abs() + tiny
        outs.append(out.flatten(1))
        tols.append(tol.flatten(1))
    return torch.cat(outs), torch.cat(tols)


def check(c, ctx, tiny=0.0):
    got = c.run(ctx).double()
    want, tol = bound(c, tiny)
    off = (got - want).abs()
    assert bool((off <= tol).all()), f"{float((off / tol.clamp_min(1e-300)).max()):.3g} of the tolerance"
    return c.out


def rows(c, seed=7, sizes=None):
    """Value rows of order one, times `sizes` [n] or [n, groups]."""
    n = c.lens[0]
    x = np.random.default_rng(seed).standard_normal((n, c.kv_heads, c.d // 32, 32))
    x /= np.abs(x).max(-1, keepdims=True)
    if sizes is not None:
        sizes = np.asarray(sizes, np.float64)
        x *= sizes[:, None, None, None] if sizes.ndim == 1 else sizes[:, None, :, None]
    return x.reshape(n, -1)


# layouts and new tokens of both kinds of tile, of every head_dim
FORMS = [("pairs", [3]), ("group_40", [3]), ("group_8", [2]), ("group_8", [70]), ("group_5", [2]), ("group_5", [30]), ("wide", [3]),
         ("wide", [40]), ("latent", [1]), ("latent", [4]), ("latent_16", [1, ]), ("latent_256", [3]), ("latent_64", [50])]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("power", [12, 24, 40, 100])
@pytest.mark.parametrize("layout,q", [f for f in FORMS if f[1][0] > 1])
def test_a_large_row_that_a_later_token_sees(ctx, layout, q, power, bf16):
    """The last token's own row is 2^power of the others: the tokens before it
    get what they get without it, but for rounding where the row is past what
    the f16 products hold."""
    c = Case(q, [130], *LAYOUTS[layout], bf16, page=64, q_scale=1.0)
    x = rows(c) * (2.0 ** -power if c.latent else 1.0)  # latent rows are keys: the large one is of order one
    plane = len(c.cache.planes) - 1
    c.cache.fill(plane, c.slots[0], x)
    without = check(c, ctx)[:-1].clone()
    x[-1] *= 2.0 ** power
    c.cache.fill(plane, c.slots[0], x)
    c.out.fill_(7.0)
    got = check(c, ctx)
    if power <= 24 and not c.latent:
        assert torch.equal(got[:-1], without)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout,q", [f for f in FORMS if not f[0].startswith("latent")])
def test_large_rows_of_no_weight(ctx, layout, q, bf16):
    """Rows of 2^30 whose scores are 60 powers of two below the others."""
    c = Case(q, [130], *LAYOUTS[layout], bf16, page=64, q_scale=0.0)
    c.q[:, :c.heads * c.d] = 1.0
    few = np.arange(130) % 5 == 2
    k = 0.1 * np.random.default_rng(4).standard_normal((130, c.kv_heads * c.d))
    k[few] = -6.0 if c.d == 64 else -4.0 if c.d == 128 else -3.0 if c.d == 256 else -2.0  # scores of about -45 and less
    c.cache.fill(0, c.slots[0], k)
    c.cache.fill(1, c.slots[0], rows(c, sizes=np.where(few, 2.0 ** 30, 1.0)))
    check(c, ctx)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("power", [9, 12, 14, 25, 60])
@pytest.mark.parametrize("layout,q", FORMS)
def test_groups_of_a_row_far_apart(ctx, layout, q, power, bf16):
    """Output dims do not add up with each other: a group of 32 dims keeps its
    bits beside one that is 2^power of it, whichever rows hold which."""
    c = Case(q, [130], *LAYOUTS[layout], bf16, page=64, q_scale=1.0)
    rng = np.random.default_rng(power)
    sizes = np.exp2(-power * rng.integers(0, 2, (130, c.d // 32)).astype(float))
    sizes[:, 0] = 2.0 ** -power  # one group is small in every row
    c.cache.fill(len(c.cache.planes) - 1, c.slots[0], rows(c, sizes=sizes))
    check(c, ctx)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout,q", [("group_8", [3]), ("group_8", [70]), ("latent_256", [3]), ("wide", [2]), ("pairs", [3])])
def test_zero_groups_and_rows_are_not_far_apart(ctx, layout, q, bf16):
    """Groups and rows of zeros, whose scale byte is 0, are of no size."""
    c = Case(q, [130], *LAYOUTS[layout], bf16, page=64, q_scale=1.0)
    sizes = np.random.default_rng(2).integers(0, 2, (130, c.d // 32)).astype(float)
    sizes[::7] = 0.0
    c.cache.fill(len(c.cache.planes) - 1, c.slots[0], rows(c, sizes=sizes))
    check(c, ctx)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout", ["group_8", "latent", "group_5"])
def test_sizes_far_apart_in_split_lists(ctx, layout, bf16):
    """A part of a long list holds values far from the others': parts of both
    kinds are joined, with a sink, with a window and without."""
    for window in (0, 2000):
        c = Case([2], [3000], *LAYOUTS[layout], bf16, page=64, q_scale=1.0, sink=True, window=window, first=3 if window else 0)
        sizes = np.ones((3000, c.d // 32))
        sizes[2100:2110, 1::2] = 2.0 ** -30
        sizes[1500] = 2.0 ** -20
        c.cache.fill(len(c.cache.planes) - 1, c.slots[0], rows(c, sizes=sizes))
        check(c, ctx)


@pytest.mark.parametrize("layout,q,lens", [("group_8", [1], [9001]), ("latent", [1, 2], [3000, 500]), ("group_8", [80], [2000]),
                                           ("pairs", [1], [6000]), ("wide", [3], [4000])])
def test_f32_sums_keep_f32(ctx, layout, q, lens):
    """Long lists in f32, whose worst-case bound would hide a weight of half as
    many bits: the rms error stays below 2e-6 of the outputs' (33 u: scores of
    up to 16 in powers of two round by 2^-21, d products by some 20 u); one f16
    part for the weights gives 2^-13 over the root of the keys that count, 1e-5."""
    c = Case(q, lens, *LAYOUTS[layout], False, page=64, q_scale=1.0)
    got = c.run(ctx).double()
    want, _ = c.expect()
    assert float((got - want).square().mean().sqrt() / want.square().mean().sqrt()) < 2e-6


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout,q,n", [("group_8", [2], 130), ("group_8", [70], 130), ("group_8", [1], 4000), ("group_5", [2], 2500),
                                        ("group_5", [40], 2500), ("pairs", [1], 1), ("pairs", [1], 6000), ("wide", [1], 3000)])
def test_values_at_the_upper_end(ctx, layout, q, n, bf16):
    """Finite values of up to 1.5 * 2^127 give finite outputs, in one part and
    joined from many."""
    for power in (125, 127.58):
        c = Case([min(q[0], n)], [n], *LAYOUTS[layout], bf16, page=64, q_scale=0.1, sink=n == 130)
        x = np.abs(rows(c)) if n > 130 else rows(c)  # of one sign, the sums stay that large
        c.cache.fill(1, c.slots[0], x * 2.0 ** power)
        check(c, ctx)
        assert bool(torch.isfinite(c.out).all())


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout,q,n", [("group_8", [2], 130), ("group_8", [70], 130), ("group_8", [1], 4000), ("group_5", [2], 2500)])
def test_values_at_the_lower_end(ctx, layout, q, n, bf16):
    """Values of some 2^-100: outputs keep f32's relative precision down to
    products of 2^-126 (n roundings of 2^-149 below)."""
    c = Case(q, [n], *LAYOUTS[layout], bf16, page=64, q_scale=0.1)
    c.cache.fill(1, c.slots[0], rows(c) * 2.0 ** -100)
    check(c, ctx, tiny=2 * n * 2.0 ** -149)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("power", [14, 23, 30, 60, 100])
@pytest.mark.parametrize("layout,q", [f for f in FORMS if not f[0].startswith("latent")])
def test_keys_and_queries_far_apart(ctx, layout, q, power, bf16):
    """Queries that are small where keys are large: a score's terms are of one
    size, whatever the factors' are.  Queries' groups are 2^power apart, keys'
    the other way round, in every third key."""
    c = Case(q, [130], *LAYOUTS[layout], bf16, page=64, q_scale=1.0)
    G, d = c.heads // c.kv_heads, c.d
    big = np.zeros(d // 32, bool)
    big[::2] = True
    up = torch.from_numpy(np.where(big, 2.0 ** -power, 1.0).repeat(32)).cuda()
    x = (c.q.double().reshape(-1, c.heads, d) * up).to(c.q.dtype)
    c.q.copy_(x.reshape(c.q.shape))
    sizes = np.where(big[None] & (np.arange(130) % 3 == 0)[:, None], 2.0 ** power, 1.0)
    c.cache.fill(0, c.slots[0], rows(c, seed=9, sizes=sizes))
    check(c, ctx)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("power", [-122, -110, 110, 124])
@pytest.mark.parametrize("layout,q", [f for f in FORMS if not f[0].startswith("latent")])
def test_queries_at_both_ends(ctx, layout, q, power, bf16):
    """Queries of 2^power and keys of 2^-power: scores of order one and ten."""
    c = Case(q, [130], *LAYOUTS[layout], bf16, page=64, q_scale=1.0)
    c.q[-1] = c.q[-1].abs()  # a query that all keys with it are large for
    c.q.copy_((c.q.double() * 2.0 ** power).to(c.q.dtype))
    k = rows(c, seed=9)
    k[::5] = np.abs(k[::5])
    c.cache.fill(0, c.slots[0], k * 2.0 ** -power)
    check(c, ctx)


@pytest.mark.parametrize("scale", [2.0 ** 90, 2.0 ** -60])
@pytest.mark.parametrize("layout,q", [("pairs", [3]), ("group_8", [2]), ("group_8", [70]), ("wide", [3])])
def test_scales_that_undo_the_sizes(ctx, layout, q, scale):
    """Queries, keys and the scale far from one, scores not, in f32."""
    c = Case(q, [130], *LAYOUTS[layout], False, page=64, q_scale=1.0)
    c.q.mul_(2.0 ** (-30 if scale > 1 else -58))
    c.cache.fill(0, c.slots[0], rows(c, seed=9) * 2.0 ** (-60 if scale > 1 else 116))
    c.scale = scale
    check(c, ctx)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout,q,n", [("pairs", [3], 130), ("group_8", [2], 130), ("group_8", [70], 130), ("group_5", [30], 130),
                                        ("wide", [3], 130), ("group_8", [1], 4000), ("group_5", [40], 2500)])
def test_scores_at_the_lower_end(ctx, layout, q, n, bf16):
    """Scores of some -2^122 are scores: the key that has the largest takes all
    of the weight."""
    c = Case(q, [n], *LAYOUTS[layout], bf16, page=64, q_scale=0.0)
    c.scale = 1.0
    c.q[:, :c.heads * c.d] = 2.0 ** 60
    k = np.full((n, c.kv_heads * c.d), -2.0 ** 56)
    k[17] = -2.0 ** 55
    c.cache.fill(0, c.slots[0], k)
    c.cache.fill(1, c.slots[0], rows(c))
    got = c.run(ctx).double()
    v = torch.from_numpy(c.cache.rows(1, c.slots[0][17:18])[0]).cuda()
    want = v.repeat_interleave(c.heads // c.kv_heads, 0).reshape(1, -1)
    assert bool(((got - want).abs() <= 4 * U * want.abs()).all())


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("layout,q", FORMS)
def test_queries_that_are_not_finite(ctx, layout, q, value, bf16):
    """They make their own head of their own token NaN."""
    c = Case(q, [300], *LAYOUTS[layout], bf16, page=64, sink=True)
    want = c.run(ctx).clone().reshape(-1, c.heads, c.d)
    c.q[-1, (c.heads // 2) * c.d + 5] = value
    c.out.fill_(7.0)
    got = c.run(ctx).reshape(-1, c.heads, c.d)
    nan = torch.zeros(len(got), c.heads, dtype=torch.bool, device="cuda")
    nan[-1, c.heads // 2] = True
    assert bool(torch.isnan(got[nan]).all()) and torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout", ["group_8", "latent_64"])
def test_a_prompt_among_single_tokens(ctx, layout, bf16):
    """One prompt of 2000 tokens beside 95 requests of one: one call, any mix."""
    q = [1] * 50 + [2000] + [1] * 45
    lens = [1 + (b * 37) % 900 for b in range(50)] + [2100] + [1 + (b * 53) % 700 for b in range(45)]
    Case(q, lens, *LAYOUTS[layout], bf16, page=16, behind=5).check(ctx)


@pytest.mark.parametrize("layout,q", [("pairs", [3]), ("group_8", [2]), ("group_8", [70]), ("group_5", [30]), ("wide", [3]), ("latent", [1])])
def test_query_groups_far_apart(ctx, layout, q):
    """f32 queries that are 2^40 larger in a group of 32 dims where the keys are
    zero: the other groups make the scores."""
    c = Case(q, [130], *LAYOUTS[layout], False, page=64, q_scale=1.0)
    up = torch.ones(c.heads * c.d, device="cuda").reshape(c.heads, c.d)
    up[:, 32:64] = 2.0 ** 40
    c.q.mul_(up.reshape(-1))
    sizes = np.ones((130, c.d // 32))
    sizes[:, 1] = 0.0
    c.cache.fill(0, c.slots[0], rows(c, seed=9, sizes=sizes))
    check(c, ctx)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("layout,q", [("pairs", [3]), ("group_8", [2]), ("group_8", [70]), ("group_5", [30]), ("wide", [3]), ("latent", [1]),
                                      ("latent_16", [1]), ("latent_256", [3]), ("latent_64", [50])])
def test_scale_byte_0(ctx, layout, q, bf16):
    """A group whose byte is 0 stands for zeros, whatever its codes: in rows
    read, in scores of queries of 2^125, in values."""
    for size in (1.0, 2.0 ** -60):  # products of f16, and the plain way
        c = Case(q, [100], *LAYOUTS[layout], bf16, page=64, q_scale=1.0)
        for k in range(len(c.cache.planes)):
            c.cache.fill(k, c.slots[0], rows(c, seed=k) * (size if k else 1.0))
        for codes, scales in c.cache.planes:
            scales[..., 1] = 0
        up = torch.ones(c.heads, c.d, device="cuda")
        up[:, 32:64] = 2.0 ** 123
        c.q.copy_((c.q.double() * up.reshape(-1)).to(c.q.dtype))
        check(c, ctx)
    slots = torch.from_numpy(c.slots[0].astype(np.int32)).cuda()
    width = c.kv_heads * c.d
    out = torch.full((100, width), 7.0, dtype=c.dt, device="cuda")
    torch.cuda.synchronize()
    ctx.kv4_read_async(c.cache.c, ptr(slots), 100, ptr(out), width, None, 0, bf16)
    ctx.synchronize()
    assert np.array_equal(out.double().cpu().numpy(), c.cache.rows(0, c.slots[0]).reshape(100, -1))
