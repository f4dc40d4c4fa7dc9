"""The 8-bit products of many positions that this library is measured on.

Five operators, each case one pass through public entry points of
wohper_amd.Context:

  quant    rows of activations (or SwiGLU of gate and up rows) rounded to 8-bit
           rows, and read back as the values they now stand for
  mm       8-bit rows times a resident FP8 weight
  groups   8-bit rows, grouped by expert, times each expert's own rows of a
           resident FP8 weight
  plan     expert lists from the routes of a batch of positions
  combine  each position's weighted sum of its experts' rows

An 8-bit row holds E4M3 codes, with one UE8M0 scale byte for every 128
columns.  Inside a block of 128 the codes lie in the weight store's order:
byte 16 l + i is column 16 (i % 8) + 8 (i / 8) + l.
"""
import math

import torch

own = False

BLOCK = 128
NONE = -1  # 0xFFFFFFFF: a route to no expert, a slot of no row


def listed():
    return [
        # activations of a few verified positions, in f32: the smallest call, where latency counts
        dict(name="quant_16", kind="quant", n=16, cols=4096, bf16=False, swiglu=False),
        # a prompt's activations before its projections
        dict(name="quant_8192", kind="quant", n=8192, cols=4096, bf16=True, swiglu=False),
        # gate and up rows of a prompt's routed positions before the down products
        dict(name="swiglu_24001", kind="quant", n=24001, cols=2048, bf16=True, swiglu=True),
        # speculative verify: five positions through the output projection
        dict(name="mm_5", kind="mm", n=5, rows=4096, cols=8192, first=0, bf16=False, f32_scales=False),
        # a short prompt through the query projection, f32 scales
        dict(name="mm_333", kind="mm", n=333, rows=32768, cols=1024, first=0, bf16=False, f32_scales=True),
        # a long prompt's chunk through the output projection
        dict(name="mm_4096", kind="mm", n=4096, rows=4096, cols=8192, first=0, bf16=True, f32_scales=False),
        # a decode step of sixteen requests: gate and up of many experts with a few positions each
        dict(name="groups_16", kind="groups", npos=16, topk=6, experts=64, rows=4096, cols=4096, gather=True, bf16=False,
             f32_scales=False),
        # a prompt's routed positions, unevenly spread, through the experts' gate and up
        dict(name="groups_4000", kind="groups", npos=4000, topk=6, experts=64, rows=4096, cols=4096, gather=True,
             bf16=True, f32_scales=False),
        # the expert lists of that decode step
        dict(name="plan_16", kind="plan", npos=16, topk=6, experts=256),
        # and of a long prompt, an eighth of it padding
        dict(name="plan_16384", kind="plan", npos=16384, topk=6, experts=256),
        # the decode step's sum over its experts
        dict(name="combine_16", kind="combine", npos=16, topk=6, hidden=4096, bf16=False),
        # a prompt's
        dict(name="combine_4000", kind="combine", npos=4000, topk=6, hidden=4096, bf16=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "quant", "mm", "mm", "mm", "groups", "groups", "groups", "plan", "combine"])
    bf16 = rng.random() < 0.5
    if kind == "quant":
        swiglu = rng.random() < 0.5
        cols = BLOCK * _log_int(rng, 1, 64)
        return dict(kind=kind, n=_log_int(rng, 1, min(24001, 40000000 // cols)), cols=cols, bf16=bf16, swiglu=swiglu)
    if kind == "plan":
        return dict(kind=kind, npos=_log_int(rng, 1, 16384), topk=rng.randint(1, 8), experts=_log_int(rng, 4, 256))
    if kind == "combine":
        return dict(kind=kind, npos=_log_int(rng, 1, 4000), topk=rng.randint(1, 8), hidden=4 * _log_int(rng, 32, 1024),
                    bf16=bf16)
    if kind == "mm":
        cols = BLOCK * _log_int(rng, 1, 64)
        rows = _log_int(rng, 100, 32768)
        first = 16 * rng.randint(0, 8) if rng.random() < 0.3 else 0
        most = min(4096, 4096 * 4096 * 8192 // (rows * cols))
        return dict(kind=kind, n=_log_int(rng, 1, most), rows=rows, cols=cols, first=first, bf16=bf16,
                    f32_scales=rng.random() < 0.4)
    experts, topk = rng.choice([4, 8, 16, 32, 64]), rng.choice([1, 2, 4, 6, 8])
    cols, rows = BLOCK * _log_int(rng, 2, 32), 64 * _log_int(rng, 4, 64)
    most = min(4000, 3 * 10**11 // (rows * cols * topk))
    return dict(kind=kind, npos=_log_int(rng, 1, most), topk=topk, experts=experts, rows=rows, cols=cols,
                gather=rng.random() < 0.5, bf16=bf16, f32_scales=rng.random() < 0.4)


# ------------------------------------------------------------ inputs

class _State:
    """A case's inputs and outputs."""

    def __init__(self, case):
        self.case, self.call, self.weight = case, None, None

    def __del__(self):
        if self.weight is not None and _kept:
            _kept["ctx"].release(self.weight)


def _float(bf16):
    return torch.bfloat16 if bf16 else torch.float32


def _rows(gen, n, cols, bf16):
    """Activations of order one; some channels are much larger, as in earnest."""
    gain = torch.exp2(2.0 * torch.randn(cols, generator=gen, device="cuda").clamp(-3, 3))
    return (torch.randn(n, cols, generator=gen, device="cuda") * gain).to(_float(bf16))


def _block_order():
    """Column of each byte of a block."""
    p = torch.arange(BLOCK, device="cuda")
    return 16 * (p % 8) + 8 * (p % 16 // 8) + p // 16


def _codes(gen, n, cols):
    """E4M3 codes of normally distributed values with a block's largest near
    the type's, [n, cols] in column order."""
    v = (torch.randn(n, cols, generator=gen, device="cuda") * 110.0).clamp_(-448.0, 448.0)
    return v.to(torch.float8_e4m3fn).view(torch.uint8)


def _in_store_order(codes):
    n, cols = codes.shape
    return codes.reshape(n, cols // BLOCK, BLOCK)[:, :, _block_order()].reshape(n, cols).contiguous()


def _pad4(n):
    return -(-n // 4) * 4


def _routes(gen, npos, topk, experts):
    """[npos, topk] experts, a few of them sought after, none twice for one
    position where there are enough; one position in eight is padding."""
    liking = 0.5 * torch.randn(experts, generator=gen, device="cuda")
    noise = -torch.log(-torch.log(torch.rand(npos, experts, generator=gen, device="cuda").clamp(1e-9, 1 - 1e-7)))
    ids = (liking + noise).topk(min(topk, experts), 1).indices
    ids = torch.cat([ids, ids[:, :max(0, topk - experts)]], 1)
    if npos >= 8:
        ids[npos - npos // 8:] = NONE
    return ids.int().contiguous()


def _lists(ids, experts):
    """Plain expert lists: starts, the position of each listed assignment and
    the place of each assignment."""
    npos, topk = ids.shape
    flat = ids.reshape(-1).long()
    some = (flat >= 0) & (flat < experts)
    key = torch.where(some, flat, experts)
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device="cuda").index_add_(0, key, torch.ones_like(key))
    starts = torch.cat([counts.new_zeros(1), counts[:experts].cumsum(0)])
    rank = torch.arange(npos * topk, device="cuda")
    rows = torch.where(rank < starts[-1], order // topk, NONE)
    slots = torch.full_like(flat, NONE)
    slots[order] = torch.where(rank < starts[-1], rank, NONE)
    return starts.int(), rows.int(), slots.int().reshape(npos, topk)


def _weight(s, gen, rows, cols):
    """A weight's codes and one scale for each 128 x 128 block (64 x 128 where
    the experts' rows ask for it)."""
    c = s.case
    s.row_block = 128 if rows % 128 == 0 and c["rows"] % 128 == 0 or c["kind"] == "mm" else 64
    s.w_codes = _codes(gen, rows, cols)
    shape = (rows // s.row_block, cols // BLOCK)
    if c["f32_scales"]:
        s.w_scales = torch.exp2(-10.0 + 6.0 * torch.rand(shape, generator=gen, device="cuda"))
    else:
        s.w_scales = torch.randint(117, 124, shape, generator=gen, device="cuda", dtype=torch.uint8)


def _row_inputs(s, gen, n, cols):
    """8-bit rows as an earlier call leaves them, and their outputs."""
    s.x_codes = _in_store_order(_codes(gen, n, cols))
    s.x_scales = torch.randint(115, 125, (n, _pad4(cols // BLOCK)), generator=gen, device="cuda", dtype=torch.uint8)


def prepare(case, seed):
    c, s = case, _State(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if c["kind"] == "quant":
        n, cols = c["n"], c["cols"]
        s.x = _rows(gen, n, cols * (2 if c["swiglu"] else 1), c["bf16"])
        s.codes = torch.empty(n, cols, dtype=torch.uint8, device="cuda")
        s.scales = torch.empty(n, _pad4(cols // BLOCK), dtype=torch.uint8, device="cuda")
        s.out = torch.empty(n, cols, dtype=torch.bfloat16, device="cuda")
    elif c["kind"] == "mm":
        _weight(s, gen, -(-(c["first"] + c["rows"]) // 128) * 128, c["cols"])
        _row_inputs(s, gen, c["n"], c["cols"])
        s.out = torch.empty(c["n"], c["rows"], dtype=_float(c["bf16"]), device="cuda")
    elif c["kind"] == "groups":
        _weight(s, gen, c["experts"] * c["rows"], c["cols"])
        s.ids = _routes(gen, c["npos"], c["topk"], c["experts"])
        s.starts, s.rows, s.slots = _lists(s.ids, c["experts"])
        s.bounds = s.starts.tolist()
        s.n_listed = c["npos"] * c["topk"]  # the buffers' rows; those past the lists are left as they are
        _row_inputs(s, gen, c["npos"] if c["gather"] else s.n_listed, c["cols"])
        s.out = torch.zeros(s.n_listed, c["rows"], dtype=_float(c["bf16"]), device="cuda")
    elif c["kind"] == "plan":
        s.ids = _routes(gen, c["npos"], c["topk"], c["experts"])
        s.starts = torch.empty(c["experts"] + 1, dtype=torch.int32, device="cuda")
        s.rows = torch.empty(c["npos"] * c["topk"], dtype=torch.int32, device="cuda")
        s.slots = torch.empty_like(s.ids)
    else:
        ids = _routes(gen, c["npos"], c["topk"], 64)
        s.n_listed = c["npos"] * c["topk"]
        s.slots = _lists(ids, 64)[2]
        s.y = _rows(gen, s.n_listed, c["hidden"], c["bf16"])
        w = torch.rand(c["npos"], c["topk"], generator=gen, device="cuda") + 0.1
        s.weights = w / w.sum(1, keepdim=True)
        s.out = torch.empty(c["npos"], c["hidden"], dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    if own:
        if c["kind"] in ("mm", "groups"):
            s.weight = _context().store_fp8_device(s.w_codes.data_ptr(), *s.w_codes.shape, s.w_scales.data_ptr(),
                                                   *s.w_scales.shape, int(c["f32_scales"]))
    return s


# ------------------------------------------------------------ the framework's calls

_kept = {}


def _context():
    """One context for the whole process, as a program has."""
    import wohper_amd

    if "ctx" not in _kept:
        _kept["ctx"] = wohper_amd.Context(0)
    return _kept["ctx"]


def _make_call(s):
    """The descriptors that a program keeps for its buffers, and the pass."""
    import wohper_amd

    ctx, c = _context(), s.case
    if c["kind"] == "plan":
        args = (s.ids.data_ptr(), c["npos"], c["topk"], c["experts"], s.starts.data_ptr(), s.rows.data_ptr(),
                s.slots.data_ptr())
        out = {"starts": s.starts, "rows": s.rows, "slots": s.slots}
        return lambda: (ctx.expert_plan_async(*args), out)[1]
    if c["kind"] == "combine":
        args = (s.y.data_ptr(), c["hidden"], int(c["bf16"]), s.n_listed, s.slots.data_ptr(), s.weights.data_ptr(),
                c["npos"], c["topk"], c["hidden"], s.out.data_ptr(), c["hidden"])
        return lambda: (ctx.expert_combine_async(*args), s.out)[1]
    if c["kind"] == "quant":
        rows = wohper_amd.WhFp8Rows(s.codes.data_ptr(), s.codes.shape[1], s.scales.data_ptr(), s.scales.shape[1])
        x, n, cols, bf16, stride = s.x.data_ptr(), c["n"], c["cols"], int(c["bf16"]), s.x.shape[1]
        if c["swiglu"]:
            up = x + cols * s.x.element_size()

            def quant():
                ctx.fp8_swiglu_rows_async(x, up, stride, bf16, n, cols, 10.0, rows)
                ctx.fp8_read_rows_async(rows, n, cols, s.out.data_ptr(), cols, 1)
                return s.out
        else:
            def quant():
                ctx.fp8_quant_rows_async(x, stride, bf16, n, cols, rows)
                ctx.fp8_read_rows_async(rows, n, cols, s.out.data_ptr(), cols, 1)
                return s.out
        return quant
    rows = wohper_amd.WhFp8Rows(s.x_codes.data_ptr(), s.x_codes.shape[1], s.x_scales.data_ptr(), s.x_scales.shape[1])
    if c["kind"] == "mm":
        args = (s.weight, c["first"], c["first"] + c["rows"], rows, c["n"], s.out.data_ptr(), c["rows"], int(c["bf16"]))
        return lambda: (ctx.fp8_rows_mm_async(*args), s.out)[1]
    args = (s.weight, 0, c["rows"], c["experts"], rows, s.x_codes.shape[0], s.rows.data_ptr() if c["gather"] else None,
            s.starts.data_ptr(), s.n_listed, s.out.data_ptr(), c["rows"], int(c["bf16"]))
    return lambda: (ctx.fp8_rows_mm_groups_async(*args), s.out)[1]


# ------------------------------------------------------------ the plain forms

def _power(e):
    """2^e in f32, e an integer tensor from -126 to 127."""
    return torch.ldexp(torch.ones((), device="cuda"), e)


def _plain_quant(s):
    c = s.case
    if c["swiglu"]:
        # in 64 bits: values next to a rounding border
        g, u = s.x.double().split(c["cols"], 1)
        g = g.clamp(max=10.0)
        v = g / (1.0 + torch.exp(-g)) * u.clamp(-10.0, 10.0)
    else:
        v = s.x.double()
    v = v.float().reshape(c["n"], -1, BLOCK)
    mant, power = torch.frexp(v.abs().amax(2, keepdim=True))
    power = (power - torch.where(mant > 0.875, 8, 9)).clamp_min(-126)
    t = torch.ldexp(v, -power).to(torch.float8_e4m3fn).float()
    return torch.ldexp(t, power).reshape(c["n"], -1).bfloat16()


def _x_values(s):
    """f32 values of the 8-bit rows, in column order."""
    n, cols = s.x_codes.shape
    v = s.x_codes.view(torch.float8_e4m3fn).float().reshape(n, cols // BLOCK, BLOCK)
    v = v * _power(s.x_scales[:, :cols // BLOCK].int() - 127)[..., None]
    out = torch.empty_like(v)
    out[:, :, _block_order()] = v
    return out.reshape(n, cols)


def _w_values(s):
    rows, cols = s.w_codes.shape
    scales = s.w_scales if s.case["f32_scales"] else _power(s.w_scales.int() - 127)
    v = s.w_codes.view(torch.float8_e4m3fn).float().reshape(rows // s.row_block, s.row_block, cols // BLOCK, BLOCK)
    return (v * scales[:, None, :, None]).reshape(rows, cols)


def _plain_mm(s):
    c = s.case
    w = _w_values(s)[c["first"]:c["first"] + c["rows"]]
    return torch.matmul(_x_values(s), w.t()).to(s.out.dtype)


def _plain_groups(s):
    """Every expert's rows padded to the longest list's."""
    c = s.case
    total, most = s.bounds[-1], max(b - a for a, b in zip(s.bounds, s.bounds[1:]))
    out = torch.zeros_like(s.out)
    if not total:
        return out
    starts = s.starts.long()
    place = starts[:-1, None] + torch.arange(most, device="cuda")
    some = place < starts[1:, None]
    place = torch.where(some, place, 0)
    x = _x_values(s)
    x = x[s.rows.long()[place] if c["gather"] else place]          # [experts, most, cols]
    w = _w_values(s).reshape(c["experts"], c["rows"], c["cols"])
    y = torch.bmm(x, w.transpose(1, 2))
    out[place[some]] = y[some].to(out.dtype)
    return out


def _plain_combine(s):
    slots = s.slots.long()
    some = slots >= 0
    y = s.y[torch.where(some, slots, 0)].float()                   # [npos, topk, hidden]
    y = torch.where(some[..., None], y, 0.0)
    return (y * s.weights[..., None]).sum(1)


def run(s):
    if own:
        if s.call is None:
            s.call = _make_call(s)
        return s.call()
    kind = s.case["kind"]
    if kind == "plan":
        starts, rows, slots = _lists(s.ids, s.case["experts"])
        return {"starts": starts, "rows": rows, "slots": slots}
    return {"quant": _plain_quant, "mm": _plain_mm, "groups": _plain_groups, "combine": _plain_combine}[kind](s)


# ------------------------------------------------------------ work

def _used(c):
    """Assignments to experts, positions that have some, and how many experts a
    batch of them reaches at most."""
    pos = c["npos"] - (c["npos"] // 8 if c["npos"] >= 8 else 0)
    return pos * c["topk"], pos, min(c.get("experts", 64), pos * c["topk"])


def work(case):
    c = case
    size = 2 if c.get("bf16") else 4
    if c["kind"] == "quant":
        codes = c["n"] * (c["cols"] + c["cols"] // BLOCK)
        inputs = c["n"] * c["cols"] * size * (2 if c["swiglu"] else 1)
        return {"bytes": inputs + 2 * codes + 2 * c["n"] * c["cols"], "flops": 0}
    if c["kind"] == "mm":
        n, rows, cols = c["n"], c["rows"], c["cols"]
        return {"bytes": (n + rows) * cols + n * cols // BLOCK + rows * cols // 16384 + n * rows * size,
                "flops": 2 * n * rows * cols}
    listed_rows, pos, experts = _used(c)
    if c["kind"] == "groups":
        rows, cols = c["rows"], c["cols"]
        inputs = pos if c["gather"] else listed_rows
        return {"bytes": (experts * rows + inputs) * cols + listed_rows * rows * size, "flops": 2 * listed_rows * rows * cols}
    if c["kind"] == "plan":
        return {"bytes": 4 * (3 * c["npos"] * c["topk"] + c["experts"] + 1), "flops": 0}
    return {"bytes": listed_rows * c["hidden"] * size + c["npos"] * (c["hidden"] * 4 + 8 * c["topk"]),
            "flops": 2 * listed_rows * c["hidden"]}


# ------------------------------------------------------------ 64 bits, from the definitions

def _e4m3_values():
    """The 127 magnitudes of E4M3, by code, in f64."""
    c = torch.arange(127, device="cuda", dtype=torch.float64)
    e, m = torch.floor(c / 8), c % 8
    return torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e - 10))


def _exact_codes(codes):
    c = codes.int()
    v = _e4m3_values()[(c % 128).clamp(max=126).long()]
    return torch.where(c >= 128, -v, v)


def _exact_quant(s):
    c = s.case
    x = s.x.double()
    if c["swiglu"]:
        g, u = x[:, :c["cols"]], x[:, c["cols"]:]
        g = torch.minimum(g, torch.full_like(g, 10.0))
        x = g * torch.sigmoid(g) * torch.clamp(u, -10.0, 10.0)
    x = x.reshape(-1, BLOCK)
    top = x.abs().amax(1)
    e = torch.ceil(torch.log2(top / 448.0)).nan_to_num(neginf=0.0)
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where((top <= 224.0 * torch.exp2(e)) & (top > 0), e - 1, e).clamp_min(-126.0)[:, None]
    grid = _e4m3_values()
    t = x.abs() / torch.exp2(e)
    hi = torch.searchsorted(grid, t).clamp(1, 126)
    lo = hi - 1
    near, far = t - grid[lo], grid[hi] - t
    code = torch.where((near < far) | ((near == far) & (lo % 2 == 0)), lo, hi)
    return (torch.sign(x) * grid[code] * torch.exp2(e)).reshape(c["n"], -1)


def _exact_x(s):
    codes = s.x_codes
    cols = codes.shape[1]
    j = torch.arange(cols, device="cuda")
    at = j // 128 * 128 + j % 8 * 16 + j % 16 // 8 * 8 + j % 128 // 16  # byte of column j
    return _exact_codes(codes[:, at]) * torch.exp2(s.x_scales[:, j // 128].double() - 127.0)


def _exact_w(s, a, b):
    r = torch.arange(a, b, device="cuda") // s.row_block
    scale = s.w_scales.double() if s.case["f32_scales"] else torch.exp2(s.w_scales.double() - 127.0)
    return _exact_codes(s.w_codes[a:b]) * scale[r].repeat_interleave(BLOCK, 1)


def exact(case, seed):
    """None for expert lists, which are whole numbers."""
    c = case
    if c["kind"] == "plan":
        return None
    s = prepare(c, seed)
    if c["kind"] == "quant":
        return _exact_quant(s)
    if c["kind"] == "combine":
        out = torch.zeros(c["npos"], c["hidden"], dtype=torch.float64, device="cuda")
        for k in range(c["topk"]):
            has = s.slots[:, k] != NONE
            out[has] += s.weights[has, k].double()[:, None] * s.y[s.slots[has, k].long()].double()
        return out
    x = _exact_x(s)
    if c["kind"] == "mm":
        return x @ _exact_w(s, c["first"], c["first"] + c["rows"]).T
    out = torch.zeros(s.n_listed, c["rows"], dtype=torch.float64, device="cuda")
    for e, (a, b) in enumerate(zip(s.bounds, s.bounds[1:])):
        if b > a:
            take = x[s.rows[a:b].long()] if c["gather"] else x[a:b]
            out[a:b] = take @ _exact_w(s, e * c["rows"], (e + 1) * c["rows"]).T
    return out
