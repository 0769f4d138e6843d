"""The operators over a paged key-value cache, as measurable cases: decode attention of a batch of sequences
(with or without the accumulation of attention weights), the append of new tokens with RoPE at each
sequence's own position, and the eviction of what was attended least.

A server of many sequences keeps one pool of cache pages ([layer][slot][kv heads][128] FP16, page p = slots
p * page .. + page) and per sequence a row of page numbers, a length and, where it evicts, the accumulated
weight of every position ([layer][row][kv heads][capacity] FP32). Each step appends one token per sequence to
each layer and attends; from time to time a sequence that outgrew its budget moves its best positions of all
layers to fresh pages.

`own` false: the definitions in elementary torch operations. True: the framework's calls.
"""
import math

import torch

own = False

HEAD_DIM = 128
# the model family's RoPE (YaRN) parameters
YARN = dict(rope_dim=HEAD_DIM, original_context=16384, freq_base=1e6, factor=16.0, beta_fast=32.0, beta_slow=1.0,
            log_multiplier=1.0, q_temperature_scale=0.1)


# ---- the cases ----

def attn(rows, length, ragged, page, kv_heads=8, group=4, scored=False, empty=0):
    return {"kind": "attn", "rows": rows, "length": length, "ragged": ragged, "page": page, "kv_heads": kv_heads,
            "group": group, "scored": scored, "empty": empty}


def append(rows, tokens, length, page, kv_heads=8, group=4, scored=False, rope=True):
    return {"kind": "append", "rows": rows, "tokens": tokens, "length": length, "page": page, "kv_heads": kv_heads,
            "group": group, "scored": scored, "rope": rope, "ragged": True, "empty": 0}


def evict(layers, rows, length, budget, recent, page, kv_heads=8, ragged=False):
    return {"kind": "evict", "layers": layers, "rows": rows, "length": length, "budget": budget, "recent": recent,
            "page": page, "kv_heads": kv_heads, "ragged": ragged, "empty": 0}


def listed():
    cases = {
        # one chat on an otherwise idle server: the smallest call
        "attn_1x500": attn(1, 500, False, 16),
        # one long document: little parallel work but along the length
        "attn_1x32k": attn(1, 32768, False, 64),
        # a busy server: sequences of every length up to 4000, two of the batch's places free
        "attn_32x4000_ragged": attn(32, 4000, True, 16, empty=2),
        # a full batch of long sequences, the largest: 2 GB of cache a layer
        "attn_64x8k": attn(64, 8192, False, 64),
        # eight query heads per kv head, odd lengths, and the weights accumulated for a later eviction
        "scored_16x2500_g8": attn(16, 2500, True, 32, group=8, scored=True),
        # a single long sequence that is kept within a budget
        "scored_1x9000": attn(1, 9000, False, 64, scored=True),
        # the new tokens of one sequence and of a full batch
        "append_1": append(1, 1, 700, 16),
        "append_256": append(256, 1, 8000, 16, scored=True),
        # a prompt that was prefilled elsewhere moves into its pages (rotated there already)
        "append_prompt_2000": append(1, 2000, 2100, 64, rope=False),
        # a sequence of the 8B-shaped model (34 blocks) is halved
        "evict_34x1x4096": evict(34, 1, 4096, 2048, 256, 64),
        # a batch of the 14B-shaped model's blocks, of which the shorter sequences stay as they are
        "evict_8x16x3000_ragged": evict(8, 16, 3000, 1000, 100, 16, ragged=True),
        # a few short sequences lose a page or so
        "evict_2x4x600": evict(2, 4, 600, 560, 64, 32),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "append", "evict"))
    page = rng.choice((16, 16, 32, 64, 128, 256))
    kv_heads, group = rng.choice((8, 8, 8, 4, 2, 1)), rng.choice((4, 4, 4, 8, 2, 1, 3, 7))
    if kind == "append":
        tokens = rng.choice((1, 1, 1, log_int(rng, 2, 2000)))
        rows = log_int(rng, 1, 256 if tokens == 1 else max(1, 2000 // tokens))
        return append(rows, tokens, tokens + log_int(rng, 1, 8000 - tokens), page, kv_heads, group,
                      rng.random() < 0.5, rng.random() < 0.7)
    if kind == "evict":
        case = evict(log_int(rng, 1, 34), log_int(rng, 1, 16), log_int(rng, 40, 8192), 0, 0, page, kv_heads,
                     rng.random() < 0.5)
        # no more work than the halved 8B-shaped sequence
        while case["layers"] * case["rows"] * case["length"] * kv_heads > 34 * 4096 * 8:
            case["rows"] = max(1, case["rows"] // 2)
            case["length"] = max(40, case["length"] * 3 // 4 + 1)
        case["budget"] = rng.randint(case["length"] // 4, case["length"] - 1)
        case["recent"] = rng.randint(1, max(1, case["budget"] // 2))
        return case
    case = attn(log_int(rng, 1, 64), log_int(rng, 1, 32768), rng.random() < 0.7, page, kv_heads, group,
                rng.random() < 0.4)
    # no more cache and no more products than the largest listed case
    while case["rows"] * case["length"] * kv_heads * max(group, 4) > 64 * 8192 * 8 * 4:
        case["length"] = case["length"] * 3 // 4
    if case["rows"] > 2 and rng.random() < 0.3:
        case["empty"] = 1
    return case


# ---- sizes and work ----

def lengths_of(c):
    """Lengths of the rows, by the case alone: the first has the full length, ragged ones spread below it,
    the last `empty` have none."""
    got = []
    for r in range(c["rows"]):
        u = 1.0 if r == 0 or not c["ragged"] else (r * 0.6180339887498949) % 1.0
        got.append(max(c.get("tokens", 1), int(round(c["length"] * u))))
    for r in range(c["empty"]):
        got[-1 - r] = 0
    return got


def pages_of(n, page):
    return -(-n // page)


def evicted_rows(c):
    return [r for r, n in enumerate(lengths_of(c)) if n > c["budget"]]


def work(case):
    """Each byte once: K and V of the visible positions, queries in, outputs out, scores read and written; the
    appended vectors in and out; the kept rows in and out with all scores read and the kept ones written."""
    c = case
    row = c["kv_heads"] * HEAD_DIM * 2
    ns = lengths_of(c)
    if c["kind"] == "attn":
        heads, seen = c["kv_heads"] * c["group"], sum(ns)
        b = seen * 2 * row + 2 * c["rows"] * heads * HEAD_DIM * 2
        b += 4 * sum(pages_of(n, c["page"]) for n in ns) + 4 * c["rows"]
        if c["scored"]:
            b += 8 * seen * c["kv_heads"]
        return {"bytes": b, "flops": 4 * HEAD_DIM * heads * seen}
    if c["kind"] == "append":
        n = c["rows"] * c["tokens"]
        b = n * 4 * row + 8 * c["rows"]
        if c["rope"]:
            b += 2 * n * row * c["group"]
        if c["scored"]:
            b += 4 * n * c["kv_heads"]
        return {"bytes": b, "flops": 6 * n * HEAD_DIM // 2 * c["kv_heads"] * (c["group"] + 1) if c["rope"] else 0}
    per = [4 * ns[r] + c["budget"] * (4 * HEAD_DIM * 2 + 8) for r in evicted_rows(c)]
    return {"bytes": c["layers"] * c["kv_heads"] * sum(per) + 4 * c["rows"], "flops": 0}


# ---- states ----

class State:
    """What the program holds: the pool, the rows' pages and lengths, scores, this step's vectors."""


_backend = None


def backend():
    """The program's one backend (of this framework)."""
    global _backend
    if _backend is None:
        from graph_horizon_amd import HipBackend
        _backend = HipBackend(0)
    return _backend


def generator(seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=torch.float16):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def scatter_pages(g, ns, page, width, first=0):
    """A table [rows][width] of distinct pages in random order, from page `first` on; places past a row's
    length hold page `first`. Returns it with the number of the last page + 1."""
    need = [pages_of(n, page) for n in ns]
    order = torch.randperm(max(1, sum(need)), generator=g, device="cuda") + first
    table = torch.full((len(ns), width), first, dtype=torch.int64, device="cuda")
    at = 0
    for r, k in enumerate(need):
        table[r, :k] = order[at:at + k]
        at += k
    return table, first + max(1, at)


def inputs(c, seed):
    """A case's tensors, from the seed alone."""
    g, s = generator(seed), State()
    s.case = c
    ns = lengths_of(c)
    s.width = pages_of(max(ns), c["page"])
    capacity = s.width * c["page"]
    s.lengths = torch.tensor(ns, device="cuda", dtype=torch.int64)
    heads = c["kv_heads"] * c.get("group", 1)
    layers = c.get("layers", 1)
    if c["kind"] == "append":
        # what lies before the new tokens is a shared prefix: only the pages that are written are the rows' own
        first = [(n - c["tokens"]) // c["page"] for n in ns]
        mine, pages = scatter_pages(g, [n - f * c["page"] for n, f in zip(ns, first)], c["page"], s.width, 1)
        at = torch.arange(s.width, device="cuda")[None] - torch.tensor(first, device="cuda")[:, None]
        s.table = torch.where(at >= 0, torch.gather(mine, 1, at.clamp(min=0)), torch.zeros_like(mine))
        shape = (c["rows"], c["tokens"])
        s.q = normal(g, *shape, heads, HEAD_DIM)
        s.k, s.v = (normal(g, *shape, c["kv_heads"], HEAD_DIM) for _ in range(2))
        s.out = torch.empty_like(s.q)
        # a sequence that lost positions to an eviction stands further on than its length says
        gap = torch.randint(0, 100, (c["rows"],), generator=g, device="cuda")
        s.positions = s.lengths - c["tokens"] + gap
        s.most = max(ns) + 100
    else:
        s.table, pages = scatter_pages(g, ns, c["page"], s.width)
    if c["kind"] == "evict":
        kept = [c["budget"] if n > c["budget"] else 0 for n in ns]
        s.to_width = pages_of(c["budget"], c["page"])
        s.to_table, pages = scatter_pages(g, kept, c["page"], s.to_width, pages)
        s.to_lengths = torch.zeros(c["rows"], dtype=torch.int64, device="cuda")
        s.to_score = torch.zeros(layers, c["rows"], c["kv_heads"], s.to_width * c["page"], device="cuda")
        s.kept = torch.zeros(layers, c["rows"], c["kv_heads"], c["budget"], dtype=torch.int32, device="cuda")
        s.act = evicted_rows(c)
    if c["kind"] == "attn":
        s.q = normal(g, c["rows"], heads, HEAD_DIM)
        s.out = torch.empty_like(s.q)
    s.slots = pages * c["page"]
    cache = (layers, s.slots, c["kv_heads"], HEAD_DIM)
    s.kc, s.vc = normal(g, *cache), normal(g, *cache)
    s.score = None
    if c["kind"] == "evict" or c["scored"]:
        # accumulated weights are far from even, and some positions were never attended to
        z = normal(g, layers, c["rows"], c["kv_heads"], capacity, dtype=torch.float32)
        s.score = torch.where(z < -1.5, torch.zeros_like(z), (2 * z).exp())
    return s


def handle(t):
    from graph_horizon_amd import _ffi as F
    return F.GhBuf(t.data_ptr(), t.numel() * t.element_size(), 0, F.BUF_VIEW, 0, 0)


def paged(s, table, lengths, score):
    """The framework's handle of a paged cache."""
    from graph_horizon_amd import _ffi as F
    c = s.case
    kv = F.GhKv(handle(s.kc), handle(s.vc), F.KV_F16, c.get("layers", 1), s.slots, c["kv_heads"], HEAD_DIM, HEAD_DIM)
    return F.GhKvPaged(kv, handle(table), handle(lengths), F.GhBuf() if score is None else handle(score),
                       c["page"], table.shape[1], c["rows"])


def prepare(case, seed):
    s = inputs(case, seed)
    s.names = ("table", "lengths") + (("to_table", "to_lengths") if case["kind"] == "evict" else ())
    s.names += ("positions",) if case["kind"] == "append" else ()
    for name in s.names:  # 32-bit on the device, as the server keeps them
        setattr(s, name, getattr(s, name).to(torch.int32))
    if own:
        backend()
        s.kv = paged(s, s.table, s.lengths, s.score)
        if case["kind"] == "evict":
            s.to_kv = paged(s, s.to_table, s.to_lengths, s.to_score)
        s.buf = {n: handle(getattr(s, n)) for n in ("q", "k", "v", "out", "positions", "kept") if hasattr(s, n)}
        if case["kind"] == "append":
            from graph_horizon_amd import Yarn
            s.yarn = Yarn(**YARN)
    return s


# ---- one pass ----

def run(s):
    c = s.case
    if c["kind"] == "attn":
        (attn_own if own else attn_plain)(s)
        return {"out": s.out} if s.score is None else {"out": s.out, "score": s.score}
    if c["kind"] == "append":
        (append_own if own else append_plain)(s)
        got = {"k": s.kc, "v": s.vc}
        if c["rope"]:
            got["q"] = s.out
        if s.score is not None:
            got["score"] = s.score
        return got
    (evict_own if own else evict_plain)(s)
    return {"k": s.kc, "v": s.vc, "score": s.to_score, "lengths": s.to_lengths, "kept": s.kept}


def attn_own(s):
    c = s.case
    backend().attention_decode_paged(s.buf["out"], s.buf["q"], s.kv, c["kv_heads"] * c["group"], c["length"], 0)


def append_own(s):
    c, b = s.case, s.buf
    if c["rope"]:
        backend().rope_kv_write_paged(s.kv, b["out"], b["q"], b["k"], b["v"], c["kv_heads"] * c["group"],
                                      b["positions"], c["tokens"], s.most, s.yarn, 0)
    else:
        backend().kv_write_paged(s.kv, b["k"], b["v"], c["tokens"], 0)


def evict_own(s):
    c = s.case
    backend().kv_evict_paged(s.to_kv, s.kv, s.buf["kept"], c["budget"], c["recent"])


def slots_of(table, page, at):
    """Slots of the positions `at` [rows][n] under `table`."""
    table = table.long()
    return torch.gather(table, 1, at // page) * page + at % page


def attn_plain(s):
    """One new token per row over its pages, in 32 bits."""
    c = s.case
    rows, hk, g = c["rows"], c["kv_heads"], c["group"]
    cap = s.width * c["page"]
    at = torch.arange(cap, device="cuda")
    seen = at[None] < s.lengths[:, None]
    slots = slots_of(s.table, c["page"], at[None].expand(rows, cap))
    k = s.kc[0][slots].permute(0, 2, 3, 1).float().contiguous()  # [rows][kv heads][128][cap]
    q = s.q.view(rows, hk, g, HEAD_DIM).float()
    x = torch.matmul(q, k) * (1 / math.sqrt(HEAD_DIM))
    del k
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(seen.any(-1)[:, None, None, None], top, torch.zeros_like(top)))
    p = p / p.sum(-1, keepdim=True)
    p = torch.where(seen[:, None, None], p, torch.zeros_like(p))
    v = s.vc[0][slots].permute(0, 2, 1, 3).float().contiguous()
    v = v.masked_fill_(~seen[:, None, :, None], 0)
    s.out.copy_(torch.matmul(p, v).view(rows, hk * g, HEAD_DIM))
    if s.score is not None:
        s.score[0, :, :, :cap] += p.sum(2)


def angles():
    """YaRN's angle per position of each pair: interpolated by the factor where the pair turns slowly."""
    y = YARN
    pair = torch.arange(HEAD_DIM // 2, device="cuda", dtype=torch.float64)

    def corr(turns):
        return (y["rope_dim"] * math.log(y["original_context"] / (turns * 2 * math.pi))
                / (2 * math.log(y["freq_base"])))

    lo, hi = max(math.floor(corr(y["beta_fast"])), 0), min(math.ceil(corr(y["beta_slow"])), y["rope_dim"] - 1)
    slow = ((pair - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    freq = y["freq_base"] ** (-2 * pair / y["rope_dim"])
    return freq / y["factor"] * slow + freq * (1 - slow)


def rotated(x, pos):
    """x [rows][tokens][heads][128] with adjacent pairs turned by pos [rows][tokens] times the angles (the
    angles in 64 bits: far positions have many turns). Positions stay below the original context, where
    queries have no temperature."""
    t = (pos.double()[..., None] * angles())[:, :, None]
    cos, sin = t.cos().float(), t.sin().float()
    a, b = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).view(x.shape).half()


def append_plain(s):
    c = s.case
    step = torch.arange(c["tokens"], device="cuda")[None]
    at = s.lengths.long()[:, None] - c["tokens"] + step
    slots = slots_of(s.table, c["page"], at)
    k = s.k
    if c["rope"]:
        pos = s.positions.long()[:, None] + step
        s.out.copy_(rotated(s.q, pos))
        k = rotated(s.k, pos)
    s.kc[0, slots] = k
    s.vc[0, slots] = s.v
    if s.score is not None:
        row = torch.arange(c["rows"], device="cuda")[:, None].expand_as(at)
        s.score[0, row, :, at] = 0


def evict_plain(s):
    """By a stable sort of the scores' order as whole numbers: the recent positions before all others, those
    past the row's length after them."""
    c = s.case
    act = torch.tensor(s.act, device="cuda")
    score = s.score[:, act]
    n = s.lengths.long()[act][None, :, None, None]
    key = score.view(torch.int32).long()
    key = torch.where(key < 0, key ^ 0x7FFFFFFF, key)
    at = torch.arange(score.shape[-1], device="cuda")
    key = torch.where(at >= n - c["recent"], torch.full_like(key, 1 << 40), key)
    key = torch.where(at >= n, torch.full_like(key, -(1 << 40)), key)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :c["budget"]].sort(-1).values
    layer = torch.arange(c["layers"], device="cuda")[:, None, None, None]
    head = torch.arange(c["kv_heads"], device="cuda")[None, None, :, None]
    page = c["page"]
    row = torch.arange(len(s.act), device="cuda")[None, :, None, None]
    source = s.table.long()[act][row, best // page] * page + best % page
    j = torch.arange(c["budget"], device="cuda")
    target = (s.to_table.long()[act][:, j // page] * page + j % page)[None, :, None]
    s.kc[layer, target, head] = s.kc[layer, source, head]
    s.vc[layer, target, head] = s.vc[layer, source, head]
    s.to_score[:, act, :, :c["budget"]] = torch.gather(score, -1, best)
    s.to_lengths[act] = c["budget"]
    s.kept[:, act] = best.int()


# ---- the same in 64 bits ----

def exact(case, seed):
    s = inputs(case, seed)
    return {"attn": exact_attn, "append": exact_append, "evict": exact_evict}[case["kind"]](s)


def cells(s, r, n, table=None):
    """The slots of row r's first n positions, in order."""
    pages = (s.table if table is None else table)[r, :pages_of(n, s.case["page"])].tolist()
    p = s.case["page"]
    return torch.cat([torch.arange(x * p, x * p + p, device="cuda") for x in pages])[:n]


def exact_attn(s):
    c = s.case
    out = torch.zeros(c["rows"], c["kv_heads"], c["group"], HEAD_DIM, dtype=torch.float64, device="cuda")
    score = None if s.score is None else s.score.double()
    for r, n in enumerate(lengths_of(c)):
        if n == 0:
            continue
        at = cells(s, r, n)
        for h in range(c["kv_heads"]):
            k, v = s.kc[0, at, h].double(), s.vc[0, at, h].double()
            q = s.q[r, h * c["group"]:(h + 1) * c["group"]].double()
            w = torch.softmax(q @ k.t() / math.sqrt(HEAD_DIM), -1)
            out[r, h] = w @ v
            if score is not None:
                score[0, r, h, :n] += w.sum(0)
    out = out.view(c["rows"], -1, HEAD_DIM)
    return {"out": out} if score is None else {"out": out, "score": score}


def exact_append(s):
    c = s.case
    kc, vc = s.kc.double(), s.vc.double()
    got = {"k": kc, "v": vc}

    def turned(x, r):
        pos = torch.arange(c["tokens"], device="cuda").double() + s.positions[r].double()
        z = torch.view_as_complex(x[r].double().view(c["tokens"], -1, HEAD_DIM // 2, 2))
        z = z * torch.polar(torch.ones_like(angles()), pos[:, None] * angles())[:, None]
        return torch.view_as_real(z).reshape(c["tokens"], -1, HEAD_DIM)

    if c["rope"]:
        got["q"] = torch.stack([turned(s.q, r) for r in range(c["rows"])])
    if s.score is not None:
        got["score"] = s.score.double()
    for r, n in enumerate(lengths_of(c)):
        at = cells(s, r, n)[n - c["tokens"]:]
        kc[0, at] = turned(s.k, r) if c["rope"] else s.k[r].double()
        vc[0, at] = s.v[r].double()
        if s.score is not None:
            got["score"][0, r, :, n - c["tokens"]:n] = 0
    return got


def exact_evict(s):
    c = s.case
    if c["layers"] * len(s.act) * c["kv_heads"] > 5000:
        return None
    kc, vc = s.kc.double(), s.vc.double()
    ns = lengths_of(c)
    old, new = s.score.double(), s.to_score.double()
    kept, lengths = s.kept.clone(), s.to_lengths.to(torch.int32)
    for r in s.act:
        n, rest = ns[r], c["budget"] - c["recent"]
        lengths[r] = c["budget"]
        source, target = cells(s, r, n), cells(s, r, c["budget"], s.to_table)
        for layer in range(c["layers"]):
            for h in range(c["kv_heads"]):
                x = old[layer, r, h, :n]
                older = x[:n - c["recent"]]
                # the rest-th largest, and of those equal to it as many as there is room for, from the front
                stay = torch.ones(n, dtype=torch.bool, device="cuda")
                least = torch.sort(older, descending=True).values[rest - 1] if rest else older.new_tensor(math.inf)
                even = older == least
                stay[:n - c["recent"]] = (older > least) | (even & (even.cumsum(0) <= rest - (older > least).sum()))
                best = stay.nonzero().view(-1)
                kept[layer, r, h] = best.int()
                new[layer, r, h, :c["budget"]] = x[best]
                kc[layer, target, h] = s.kc[layer, source[best], h].double()
                vc[layer, target, h] = s.vc[layer, source[best], h].double()
    return {"k": kc, "v": vc, "score": new, "lengths": lengths, "kept": kept}
