"""The paged 4-bit attention cache that this library is measured on.

Three operators, each case one pass through public entry points of
wohper_amd.Context:

  plan    block tables, free pages, slots and positions of a serving step,
          from the requests' lengths before and after it
  write   the cache's rows: those of new tokens rounded into it, and read back
          as the values they now stand for
  read    the cache's rows: by slot, as values
  attend  attention of new tokens over their requests' cached rows, with a
          sliding window, first tokens that stay visible and sink logits

The cache holds E2M1 codes, two a byte (low nibble: the even dim), with one
UE8M0 scale byte for every 32 dims, in pages of `page` rows: codes
[page][kv head][row][head_dim / 2], scales [page][kv head][row][head_dim / 32].
`latent` rows are keys and values at once (64 heads over one row of 512, the
layout of the MLA layers); else keys and values are separate, kv_heads of each.
"""
import math

import torch

own = False

NO_SLOT = -1  # 0xFFFFFFFF


def listed():
    return [
        # a decode step of a small server: every request one token on, a few ended or cut back
        dict(name="plan_64", kind="plan", requests=64, page=64, old=32768, new=1),
        # a step that admits prompts: hundreds of requests, tens of thousands of tokens, small pages
        dict(name="plan_512", kind="plan", requests=512, page=16, old=4096, new=256),
        # the new rows of a decode step, one latent row a token, in the activations' f32
        dict(name="write_48", kind="write", n=48, kv_heads=1, head_dim=512, latent=True, bf16=False, page=64),
        # the keys and values of prompts' chunks
        dict(name="write_20011", kind="write", n=20011, kv_heads=8, head_dim=128, latent=False, bf16=True, page=16),
        # a shared prefix of a long document as f32 rows
        dict(name="read_50021", kind="read", n=50021, kv_heads=1, head_dim=512, latent=True, bf16=False, page=64),
        # one request at the start of its answer: the smallest call, where latency counts
        dict(name="attend_1", kind="attend", requests=1, q=1, context=130, heads=64, kv_heads=1, head_dim=512,
             latent=True, bf16=False, page=64, window=0, first=0, sink=True),
        # a decode step of a dozen long contexts
        dict(name="attend_latent_12", kind="attend", requests=12, q=1, context=40000, heads=64, kv_heads=1,
             head_dim=512, latent=True, bf16=True, page=64, window=0, first=0, sink=True),
        # speculative verify: a few drafted tokens a request, in f32
        dict(name="attend_verify_3", kind="attend", requests=3, q=5, context=6000, heads=64, kv_heads=1, head_dim=512,
             latent=True, bf16=False, page=64, window=0, first=0, sink=True),
        # a decode step of grouped heads: eight queries a key head, little arithmetic a byte
        dict(name="attend_grouped_32", kind="attend", requests=32, q=1, context=8192, heads=64, kv_heads=8,
             head_dim=128, latent=False, bf16=True, page=16, window=0, first=0, sink=False),
        # the same over a sliding window with four first tokens, in f32: many short key lists
        dict(name="attend_window_96", kind="attend", requests=96, q=1, context=9000, heads=32, kv_heads=8,
             head_dim=128, latent=False, bf16=False, page=16, window=1024, first=4, sink=False),
        # prompts of unequal lengths from their first token
        dict(name="attend_prompts_5", kind="attend", requests=5, q=2500, context=0, heads=32, kv_heads=8,
             head_dim=128, latent=False, bf16=True, page=16, window=0, first=0, sink=False),
        # a prompt's chunk over its latent rows so far
        dict(name="attend_chunk_384", kind="attend", requests=1, q=384, context=4000, heads=64, kv_heads=1,
             head_dim=512, latent=True, bf16=True, page=64, window=0, first=0, sink=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _layout(rng):
    if rng.random() < 0.5:
        return dict(kv_heads=1, head_dim=512, latent=True)
    return dict(kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128, 128, 256]), latent=False)


def draw(rng):
    kind = rng.choice(["plan", "write", "read", "attend", "attend", "attend", "attend", "attend"])
    page = rng.choice([8, 16, 32, 64, 64, 128, 256])
    if kind == "plan":
        return dict(kind=kind, requests=_log_int(rng, 1, 512), page=page, old=_log_int(rng, 16, 32768),
                    new=_log_int(rng, 1, 256))
    if kind != "attend":
        s = _layout(rng)
        per = s["kv_heads"] * s["head_dim"] * (1 if s["latent"] else 2)
        return dict(kind=kind, n=_log_int(rng, 1, 50000 * 512 // max(512, per)), bf16=rng.random() < 0.5, page=page, **s)
    s = _layout(rng)
    bf16 = rng.random() < 0.5
    s["heads"] = rng.choice([16, 50, 64, 64, 128]) if s["latent"] else s["kv_heads"] * rng.choice([1, 3, 4, 8, 16])
    form = rng.choice(["decode", "verify", "prompt"])
    window, first = (0, 0) if rng.random() < 0.6 else (_log_int(rng, 16, 4096), rng.choice([0, 1, 4, 16]))
    if form == "decode":
        q, context = 1, _log_int(rng, 16, 40000)
    elif form == "verify":
        q, context = rng.randint(2, 8), _log_int(rng, 16, 8000)
    else:
        q, context = _log_int(rng, 16, 1500), rng.choice([0, 0, _log_int(rng, 16, 4000)])
    # as many requests as keep the arithmetic and the rows under the largest listed case's
    seen = min(window + first, context + q) if window else context + q
    cost = 4.0 * q * seen * s["heads"] * s["head_dim"] * (1.0 if bf16 else 4.0)
    rows = float(context + q) * s["kv_heads"] * s["head_dim"]
    most = max(1, min(96, int(1.4e11 // cost), int(2.4e8 // rows)))
    return dict(kind=kind, requests=_log_int(rng, 1, most), q=q, context=context, bf16=bf16, page=page, window=window,
                first=first, sink=rng.random() < 0.5, **s)


# ------------------------------------------------------------ lengths and inputs

def _uneven(b, hi):
    """Request b's share of `hi`: between half of it and all of it."""
    return hi - int(hi * 0.5 * math.fmod(b * 0.6180339887, 1.0))


def _plan_lens(case):
    """Lengths before and after a step: most grow, one in five gives back
    three drafted tokens, one in sixteen ends."""
    old = [_uneven(b, case["old"]) for b in range(case["requests"])]
    new = [0 if b % 16 == 7 else max(0, o - 3) if b % 5 == 3 else o + _uneven(b + 1, case["new"])
           for b, o in enumerate(old)]
    return old, new


def _attend_lens(case):
    """(new tokens, cached tokens with them) of each request."""
    q = [_uneven(b, case["q"]) if case["q"] > 8 else case["q"] for b in range(case["requests"])]
    return q, [_uneven(b + 3, case["context"]) + n for b, n in enumerate(q)]


def _pages(n, page):
    return -(-n // page)


def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rows(gen, n, kv_heads, head_dim, bf16):
    """Rows of order one whose channels differ in size, as keys' do."""
    gain = torch.exp2(2.0 * torch.rand(kv_heads, head_dim, generator=gen, device="cuda") - 1.0)
    x = torch.randn(n, kv_heads, head_dim, generator=gen, device="cuda") * gain
    return (x.bfloat16() if bf16 else x).reshape(n, kv_heads * head_dim)


def _round_rows(x, kv_heads, head_dim):
    """[n, kv_heads * head_dim] as E2M1 codes [n, kv_heads, head_dim / 2] and
    scale bytes [n, kv_heads, head_dim / 32]: the least power of two under
    which the group's largest magnitude is at most 6, to nearest, ties to the
    even code."""
    x = x.float().reshape(x.shape[0], kv_heads, head_dim // 32, 32)
    top = x.abs().amax(3)
    mant, power = torch.frexp(top)
    power = (power - torch.where(mant > 0.75, 2, 3)).clamp_min(-126)
    t = torch.ldexp(x.abs(), -power[..., None])
    code = ((t > 0.25).to(torch.uint8) + (t >= 0.75) + (t > 1.25) + (t >= 1.75) + (t > 2.5) + (t >= 3.5) + (t > 5.0)
            + 8 * torch.signbit(x)).to(torch.uint8)
    byte = torch.where(top > 0, power + 127, 0).to(torch.uint8)
    code = code.reshape(x.shape[0], kv_heads, head_dim // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), byte


def _grid():
    m = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    return torch.cat([m, -m])


def _values(codes, scales):
    """Codes [..., d / 2] and scale bytes [..., d / 32] as f32 [..., d]."""
    grid = _grid()
    v = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1)
    v = v.reshape(*scales.shape, 32) * torch.ldexp(torch.ones((), device="cuda"), scales.int() - 127)[..., None]
    return v.reshape(*scales.shape[:-1], -1)


class _State:
    """A case's inputs and outputs.  Tensors named *_codes and *_scales are a
    cache; pages that no request owns hold other requests' old bytes."""

    def __init__(self, case):
        self.case, self.call = case, None


def _empty_cache(s, gen, n_pages):
    c = s.case
    shape = (n_pages, c["kv_heads"], c["page"])
    s.n_pages = n_pages

    def old_bytes(width):
        return torch.randint(0, 256, (*shape, width), generator=gen, device="cuda", dtype=torch.uint8)

    s.k_codes, s.k_scales = old_bytes(c["head_dim"] // 2), old_bytes(c["head_dim"] // 32)
    s.v_codes = s.v_scales = None
    if not c["latent"]:
        s.v_codes, s.v_scales = old_bytes(c["head_dim"] // 2), old_bytes(c["head_dim"] // 32)


def _put(s, codes, scales, x, slots):
    c = s.case
    q, b = _round_rows(x, c["kv_heads"], c["head_dim"])
    page, row = slots.long() // c["page"], slots.long() % c["page"]
    codes[page, :, row], scales[page, :, row] = q, b


def _take(s, codes, scales, slots):
    """f32 rows [..., kv_heads, head_dim] of the slots."""
    page, row = slots.long() // s.case["page"], slots.long() % s.case["page"]
    return _values(codes[page, :, row], scales[page, :, row])


def _prepare_rows(s, gen):
    c = s.case
    n, width = c["n"], c["kv_heads"] * c["head_dim"]
    n_pages = _pages(n, c["page"]) + 3
    _empty_cache(s, gen, n_pages)
    order = torch.randperm(n_pages, generator=gen, device="cuda")
    at = torch.arange(n, device="cuda") + 5 % c["page"]
    s.slots = (order[at // c["page"]] * c["page"] + at % c["page"]).int()
    s.k_rows = _rows(gen, n, c["kv_heads"], c["head_dim"], c["bf16"])
    s.v_rows = None if c["latent"] else _rows(gen, n, c["kv_heads"], c["head_dim"], c["bf16"])
    dtype = torch.bfloat16 if c["bf16"] else torch.float32
    s.k_out = torch.empty(n, width, device="cuda", dtype=dtype)
    s.v_out = None if c["latent"] else torch.empty(n, width, device="cuda", dtype=dtype)
    if c["kind"] == "read":
        _put(s, s.k_codes, s.k_scales, s.k_rows, s.slots)
        if not c["latent"]:
            _put(s, s.v_codes, s.v_scales, s.v_rows, s.slots)


def _prepare_attend(s, gen):
    c = s.case
    s.q_lens, s.lens = _attend_lens(c)
    counts = [_pages(n, c["page"]) for n in s.lens]
    n_pages, s.table_stride = sum(counts) + 2, max(counts) + 1
    _empty_cache(s, gen, n_pages)
    order = torch.randperm(n_pages, generator=gen, device="cuda").int()
    # entries past a request's pages are old ones, any page of the cache
    s.tables = torch.randint(0, n_pages, (c["requests"], s.table_stride), generator=gen, device="cuda",
                             dtype=torch.int32)
    at = 0
    for b, n in enumerate(s.lens):
        s.tables[b, :counts[b]] = order[at:at + counts[b]]
        at += counts[b]
        pos = torch.arange(n, device="cuda")
        slots = s.tables[b][pos // c["page"]].long() * c["page"] + pos % c["page"]
        _put(s, s.k_codes, s.k_scales, _rows(gen, n, c["kv_heads"], c["head_dim"], c["bf16"]), slots)
        if not c["latent"]:
            _put(s, s.v_codes, s.v_scales, _rows(gen, n, c["kv_heads"], c["head_dim"], c["bf16"]), slots)
    s.n_tokens = sum(s.q_lens)
    s.starts = _i32([sum(s.q_lens[:b]) for b in range(c["requests"] + 1)])
    s.lens_dev = _i32(s.lens)
    dtype = torch.bfloat16 if c["bf16"] else torch.float32
    # scores with a deviation of two to three: some keys stand out
    s.q = (2.0 * torch.randn(s.n_tokens, c["heads"] * c["head_dim"], generator=gen, device="cuda")).to(dtype)
    s.sink = torch.randn(c["heads"], generator=gen, device="cuda") if c["sink"] else None
    s.out = torch.empty_like(s.q)


def _prepare_plan(s, gen):
    c = s.case
    n, page = c["requests"], c["page"]
    old, new = _plan_lens(c)
    s.old, s.new = _i32(old), _i32(new)
    held = [_pages(v, page) for v in old]
    most = [max(a, _pages(v, page)) for a, v in zip(held, new)]
    s.table_stride = max(most) + 1
    s.n_pages = sum(most) + 5
    order = torch.randperm(s.n_pages, generator=gen, device="cuda").int()
    s.tables = torch.full((n, s.table_stride), NO_SLOT, dtype=torch.int32, device="cuda")
    at = 0
    for b, k in enumerate(held):
        s.tables[b, :k] = order[at:at + k]
        at += k
    s.free = torch.zeros(s.n_pages, dtype=torch.int32, device="cuda")
    s.free[:s.n_pages - at] = order[at:]
    s.n_free = s.n_pages - at
    s.free_count = _i32([s.n_free])
    s.tokens = sum(max(0, b - a) for a, b in zip(old, new))
    s.max_tokens = s.tokens + s.tokens // 8 + 8  # the step's buffers are a little longer than the step
    s.grown = sum(max(0, _pages(b, page) - h) for h, b in zip(held, new))
    s.shrunk = sum(max(0, h - _pages(b, page)) for h, b in zip(held, new))
    s.free_out, s.free_count_out = torch.zeros_like(s.free), torch.zeros_like(s.free_count)
    s.starts = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    s.slots = torch.zeros(s.max_tokens, dtype=torch.int32, device="cuda")
    s.positions = torch.zeros_like(s.slots)


def prepare(case, seed):
    s = _State(case)
    gen = _gen(seed)
    {"plan": _prepare_plan, "write": _prepare_rows, "read": _prepare_rows, "attend": _prepare_attend}[case["kind"]](s, gen)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------ the framework's calls

_kept = {}


def _context():
    """One context for the whole process, as a program has."""
    import wohper_amd

    if "ctx" not in _kept:
        _kept["ctx"] = wohper_amd.Context(0)
    return _kept["ctx"]


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _cache(s):
    import wohper_amd

    c = s.case
    return wohper_amd.WhKv4Cache(_ptr(s.k_codes), _ptr(s.k_scales), _ptr(s.v_codes), _ptr(s.v_scales), s.n_pages,
                                 c["page"], c["kv_heads"], c["head_dim"])


def _make_call(s):
    """The descriptors that a program keeps for its buffers, and the pass."""
    import wohper_amd

    ctx, c = _context(), s.case
    if c["kind"] == "plan":
        d = wohper_amd.WhKvPlan(c["requests"], _ptr(s.old), _ptr(s.new), _ptr(s.tables), s.table_stride, c["page"],
                                s.n_pages, _ptr(s.free), _ptr(s.free_count), _ptr(s.free_out), _ptr(s.free_count_out),
                                s.max_tokens, _ptr(s.starts), _ptr(s.slots), _ptr(s.positions))
        out = {"tables": s.tables, "free": s.free_out, "free_count": s.free_count_out, "starts": s.starts,
               "slots": s.slots, "positions": s.positions}
        return lambda: (ctx.kv_plan_async(d), out)[1]
    cache = _cache(s)
    if c["kind"] == "attend":
        d = wohper_amd.WhKv4Attention(_ptr(s.q), s.q.shape[1], _ptr(s.out), s.out.shape[1], int(c["bf16"]),
                                      s.n_tokens, c["requests"], _ptr(s.starts), _ptr(s.lens_dev), _ptr(s.tables),
                                      s.table_stride, max(s.lens), c["heads"], c["head_dim"] ** -0.5, c["window"],
                                      c["first"], _ptr(s.sink))
        return lambda: (ctx.kv4_attention_async(cache, d), s.out)[1]
    width, n, bf16 = c["kv_heads"] * c["head_dim"], c["n"], int(c["bf16"])
    out = {"k": s.k_out} if c["latent"] else {"k": s.k_out, "v": s.v_out}
    kr, vr, ko, vo, slots = (_ptr(t) for t in (s.k_rows, s.v_rows, s.k_out, s.v_out, s.slots))

    def rows():
        if c["kind"] == "write":
            ctx.kv4_write_async(cache, kr, width, vr, width, bf16, slots, n)
        ctx.kv4_read_async(cache, slots, n, ko, width, vo, width, bf16)
        return out

    return rows


# ------------------------------------------------------------ the plain forms

def _plain_plan(s):
    c = s.case
    page = c["page"]
    old, new = s.old.long(), s.new.long()
    po, pn = (old + page - 1) // page, (new + page - 1) // page
    grow, shrink, step = (pn - po).clamp_min(0), (po - pn).clamp_min(0), (new - old).clamp_min(0)
    b = torch.arange(c["requests"], device="cuda")

    def spread(counts, total):
        """Request and index within the request of each of `total` things."""
        req = torch.repeat_interleave(b, counts, output_size=total)
        return req, torch.arange(total, device="cuda") - (torch.cumsum(counts, 0) - counts)[req]

    # the pages that are given back go on the stack, in request order, then the new ones come off it
    req, k = spread(shrink, s.shrunk)
    free_out = torch.zeros_like(s.free)
    free_out[:s.n_free] = s.free[:s.n_free]
    free_out[s.n_free:s.n_free + s.shrunk] = s.tables[req, pn[req] + k]
    top = s.n_free + s.shrunk
    req, k = spread(grow, s.grown)
    tables = s.tables.clone()
    tables[req, po[req] + k] = free_out[top - 1 - torch.arange(s.grown, device="cuda")]
    req, k = spread(step, s.tokens)
    pos = old[req] + k
    slots = torch.full_like(s.slots, NO_SLOT)
    positions = torch.zeros_like(s.positions)
    slots[:s.tokens] = (tables[req, pos // page] * page + pos % page).int()
    positions[:s.tokens] = pos.int()
    starts = torch.zeros_like(s.starts)
    starts[1:] = torch.cumsum(step, 0)
    return {"tables": tables, "free": free_out, "free_count": s.free_count + (s.shrunk - s.grown), "starts": starts,
            "slots": slots, "positions": positions}


def _plain_attend(s):
    """Every request padded to the longest: [request, kv head, its queries,
    its visible keys], all in f32."""
    c = s.case
    n, kv, d = c["requests"], c["kv_heads"], c["head_dim"]
    group, width = c["heads"] // kv, max(s.q_lens)
    lens, starts = s.lens_dev.long(), s.starts.long()
    q_lens = starts[1:] - starts[:-1]
    first_pos = lens - q_lens
    i = torch.arange(width, device="cuda")
    rows = torch.minimum(starts[:-1, None] + i, torch.tensor(s.n_tokens - 1, device="cuda"))
    pos = first_pos[:, None] + i                                     # [n, width]
    q = s.q.float().reshape(s.n_tokens, kv, group, d)[rows]          # [n, width, kv, group, d]
    q = q.permute(0, 2, 1, 3, 4).reshape(n, kv, width * group, d)
    # keys: the first tokens, then from the first query's window on
    if c["window"]:
        lo = (first_pos - c["window"] + 1).clamp_min(c["first"])
        span = min(max(s.lens), c["first"] + c["window"] + width - 1)
        j = torch.arange(span, device="cuda")
        key = torch.where(j < c["first"], j, lo[:, None] + j - c["first"])
    else:
        key = torch.arange(max(s.lens), device="cuda").expand(n, -1)
    inside = key < lens[:, None]
    safe = torch.where(inside, key, 0)
    page = torch.gather(s.tables.long(), 1, safe // c["page"])
    slots = torch.where(inside, page * c["page"] + safe % c["page"], s.tables[:, :1].long() * c["page"])
    k = _take(s, s.k_codes, s.k_scales, slots).permute(0, 2, 1, 3)   # [n, kv, keys, d]
    v = k if c["latent"] else _take(s, s.v_codes, s.v_scales, slots).permute(0, 2, 1, 3)
    seen = inside[:, None] & (key[:, None] <= pos[:, :, None])       # [n, width, keys]
    if c["window"]:
        seen &= (key[:, None] > pos[:, :, None] - c["window"]) | (key[:, None] < c["first"])
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
    scores = scores.reshape(n, kv, width, group, -1)
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    sink = s.sink.reshape(kv, 1, group, 1) if c["sink"] else None
    if sink is not None:
        top = torch.maximum(top, sink)
    w = torch.exp(scores.sub_(top))
    total = w.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    out = torch.matmul(w.reshape(n, kv, width * group, -1), v).reshape(n, kv, width, group, d) / total
    out = out.permute(0, 2, 1, 3, 4).reshape(n, width, c["heads"] * d)
    req = torch.repeat_interleave(torch.arange(n, device="cuda"), q_lens, output_size=s.n_tokens)
    return out[req, torch.arange(s.n_tokens, device="cuda") - starts[req]].to(s.q.dtype)


def run(s):
    if own:
        if s.call is None:
            s.call = _make_call(s)
        return s.call()
    c = s.case
    if c["kind"] == "plan":
        return _plain_plan(s)
    if c["kind"] == "attend":
        return _plain_attend(s)
    if c["kind"] == "write":
        _put(s, s.k_codes, s.k_scales, s.k_rows, s.slots)
        if not c["latent"]:
            _put(s, s.v_codes, s.v_scales, s.v_rows, s.slots)
    n = c["n"]
    out = {"k": _take(s, s.k_codes, s.k_scales, s.slots).reshape(n, -1).to(s.k_out.dtype)}
    if not c["latent"]:
        out["v"] = _take(s, s.v_codes, s.v_scales, s.slots).reshape(n, -1).to(s.k_out.dtype)
    return out


# ------------------------------------------------------------ work

def work(case):
    c = case
    if c["kind"] == "plan":
        old, new = _plan_lens(c)
        moved = sum(abs(_pages(b, c["page"]) - _pages(a, c["page"])) for a, b in zip(old, new))
        tokens = sum(max(0, b - a) for a, b in zip(old, new))
        return {"bytes": 4 * (3 * c["requests"] + 2 * moved + 2 * tokens), "flops": 0}
    planes = 1 if c["latent"] else 2
    row = planes * c["kv_heads"] * (c["head_dim"] // 2 + c["head_dim"] // 32)
    size = 2 if c["bf16"] else 4
    if c["kind"] != "attend":
        values = planes * c["kv_heads"] * c["head_dim"] * size
        passes = 2 if c["kind"] == "write" else 1  # rows in and codes out, codes in and values out
        return {"bytes": c["n"] * (passes * (row + values) + 4 * passes), "flops": 0}
    q, lens = _attend_lens(c)
    pairs = keys = 0
    for n, m in zip(q, lens):
        w, f = c["window"], c["first"]
        if not w:
            pairs += n * m - n * (n - 1) // 2
            keys += m
        else:
            # a query at p sees min(p + 1, window) rows and those of the first ones that are before them
            pairs += sum(min(p + 1, w) + min(f, max(0, p + 1 - w)) for p in range(m - n, m))
            keys += min(m, w + n - 1) + min(f, max(0, m - n + 1 - w))
    return {"bytes": keys * row + 2 * sum(q) * c["heads"] * c["head_dim"] * size,
            "flops": 4 * pairs * c["heads"] * c["head_dim"]}


# ------------------------------------------------------------ 64 bits, from the definitions

def _exact_rows(x, heads, d):
    """Each value to the nearest of its group's sixteen, by distance; of two
    as near the one with the even code."""
    x = x.double().reshape(-1, heads, d // 32, 32)
    top = x.abs().amax(3, keepdim=True)
    scale = torch.ones_like(top)
    for _ in range(200):  # least power of two with top <= 6 * scale
        scale = torch.where(top > 6 * scale, scale * 2, scale)
        scale = torch.where((top <= 3 * scale) & (top > 0), scale / 2, scale)
    scale = torch.where(top > 6 * scale, scale * 2, scale)
    t = x.abs() / scale
    best, dist = torch.zeros_like(t), t.clone()
    for code, m in enumerate([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], start=1):
        e = (t - m).abs()
        closer = (e < dist) | ((e == dist) & (code % 2 == 0))
        best, dist = torch.where(closer, m, best), torch.minimum(e, dist)
    return (torch.sign(x) * best * scale).reshape(-1, heads * d)


def _exact_attend(case, seed):
    c = case
    s = prepare(case, seed)
    n, kv, d = c["requests"], c["kv_heads"], c["head_dim"]
    group = c["heads"] // kv
    half = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], device="cuda", dtype=torch.float64) / 2
    outs, at = [], 0

    def rows(codes, scales, b, where, h):
        """f64 [keys, d] of kv head h."""
        page, r = s.tables[b].long()[where // c["page"]], where % c["page"]
        byte, e = codes[page, h, r].long(), scales[page, h, r].double()
        nib = torch.stack([byte % 16, byte // 16], 2).reshape(len(where), d)
        v = half[nib % 8] * (1 - 2 * (nib // 8)).double()
        return v * torch.exp2(e - 127.0).repeat_interleave(32, 1)

    for b in range(n):
        nq, m = s.q_lens[b], s.lens[b]
        out = torch.empty(nq, c["heads"], d, device="cuda", dtype=torch.float64)
        for i0 in range(0, nq, 256):
            i1 = min(nq, i0 + 256)
            p = torch.arange(m - nq + i0, m - nq + i1, device="cuda")
            j = torch.arange(m, device="cuda")
            if c["window"]:
                j = j[(j < c["first"]) | (j > m - nq + i0 - c["window"])]
            hidden = j[None] > p[:, None]
            if c["window"]:
                hidden |= (j[None] <= p[:, None] - c["window"]) & (j[None] >= c["first"])
            for h in range(kv):
                k = rows(s.k_codes, s.k_scales, b, j, h)
                v = k if c["latent"] else rows(s.v_codes, s.v_scales, b, j, h)
                q = s.q[at + i0:at + i1].double().reshape(i1 - i0, c["heads"], d)[:, h * group:(h + 1) * group]
                sc = (q.reshape(-1, d) @ k.T).reshape(i1 - i0, group, -1) / math.sqrt(d)
                sc = sc.masked_fill(hidden[:, None], -math.inf)
                if c["sink"]:
                    extra = s.sink[h * group:(h + 1) * group].double()[None, :, None].expand(i1 - i0, -1, 1)
                    w = torch.softmax(torch.cat([sc, extra], 2), 2)[..., :-1]
                else:
                    w = torch.softmax(sc, 2)
                out[i0:i1, h * group:(h + 1) * group] = (w.reshape(-1, len(j)) @ v).reshape(i1 - i0, group, d)
        outs.append(out.reshape(nq, -1))
        at += nq
    return torch.cat(outs)


def exact(case, seed):
    """None for a plan, whose outputs are whole numbers."""
    if case["kind"] == "plan":
        return None
    if case["kind"] == "attend":
        return _exact_attend(case, seed)
    s = prepare(dict(case, kind="write"), seed)
    out = {"k": _exact_rows(s.k_rows, case["kv_heads"], case["head_dim"])}
    if not case["latent"]:
        out["v"] = _exact_rows(s.v_rows, case["kv_heads"], case["head_dim"])
    return out
