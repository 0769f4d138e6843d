"""A decode step of a batch of sequences whose key-value cache is held in 4 bits, as measurable cases: norms of
queries and keys per head with the position rotation (alone, or on the way into the cache), the append to a paged
4-bit cache, attention over it, and the draw of each row's next token from its logits.

A pool of pages as of the FP16 operators, with 80 bytes per vector of 128 values: 64 bytes of codes, dims 2 i and
2 i + 1 in the low and high half of byte i, then for each 32 dims a step d and a minimum m in FP16. A code c stands
for m + d c. Of 32 values, m is the least one in FP16 and d a fifteenth of their range, cut off to FP16; the code is
(x - m) / d as the nearest whole number (ties to even), 0 to 15.

`own` false: the definitions in elementary torch operations. True: the framework's calls.
"""
import math

import numpy as np
import torch

own = False

HEAD_DIM = 128
VECTOR = 80  # bytes
EPS = 1e-5
# the model family's RoPE (YaRN) parameters
YARN = dict(rope_dim=HEAD_DIM, original_context=16384, freq_base=1e6, factor=16.0, beta_fast=32.0, beta_slow=1.0,
            log_multiplier=1.0, q_temperature_scale=0.1)


# ---- the cases ----

def attn(rows, length, ragged, page, kv_heads=8, group=4, scored=False, empty=0):
    return {"kind": "attn", "rows": rows, "length": length, "ragged": ragged, "page": page, "kv_heads": kv_heads,
            "group": group, "scored": scored, "empty": empty}


def append(rows, tokens, length, page, kv_heads=8, group=4, scored=False, form="norm", bits=4):
    """form: "norm" (norms and rotation), "rope" (rotation alone), "plain" (neither; no queries)."""
    return {"kind": "append", "rows": rows, "tokens": tokens, "length": length, "page": page, "kv_heads": kv_heads,
            "group": group, "scored": scored, "form": form, "bits": bits, "ragged": True, "empty": 0}


def norm(rows, base, kv_heads=8, group=4, head_dim=HEAD_DIM):
    return {"kind": "norm", "rows": rows, "base": base, "kv_heads": kv_heads, "group": group, "head_dim": head_dim}


def sample(rows, vocab, top_k, top_p, min_p, temperature, mixed=False):
    """mixed: each row with settings of its own around these, some greedy, some without a filter."""
    return {"kind": "sample", "rows": rows, "vocab": vocab, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "temperature": temperature, "mixed": mixed}


def listed():
    cases = {
        # one chat on an otherwise idle server: the smallest call
        "attn_1x500": attn(1, 500, False, 16),
        # a busy server: sequences of every length up to 4000, two of the batch's places free
        "attn_32x4000_ragged": attn(32, 4000, True, 16, empty=2),
        # a full batch of long sequences, the largest
        "attn_64x8k": attn(64, 8192, False, 64),
        # eight query heads per kv head, odd lengths, and the weights accumulated for a later eviction
        "scored_16x2500_g8": attn(16, 2500, True, 32, group=8, scored=True),
        # the new token of one sequence and of a full batch
        "append_1": append(1, 1, 700, 16),
        "append_256": append(256, 1, 8000, 16, scored=True),
        # a prompt that was prefilled elsewhere moves into its pages (normed and rotated there already)
        "append_prompt_2000": append(1, 2000, 2100, 64, form="plain"),
        # norms and rotation before prefill attention: a chunk of a long prompt, and one token
        "norm_2000": norm(2000, 6000),
        "norm_1": norm(1, 519),
        # one chat's next token, by the usual settings
        "sample_1": sample(1, 131072, 50, 0.9, 0.0, 0.8),
        # a full batch, each request with settings of its own
        "sample_64_mixed": sample(64, 131072, 40, 0.95, 0.05, 0.9, mixed=True),
        # a few rows by top-p alone, which looks at the whole vocabulary
        "sample_8_top_p": sample(8, 131072, 0, 0.97, 0.0, 1.2),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("attn", "attn", "append", "append", "norm", "sample", "sample"))
    page = rng.choice((16, 16, 32, 64, 128, 256))
    kv_heads, group = rng.choice((8, 8, 8, 4, 2, 1)), rng.choice((4, 4, 4, 8, 2, 1, 3, 7))
    if kind == "norm":
        return norm(log_int(rng, 1, 2000), rng.randint(0, 30000), kv_heads, min(group, 4), rng.choice((128, 128, 64)))
    if kind == "sample":
        return sample(log_int(rng, 1, 64), log_int(rng, 1000, 131072), rng.choice((0, log_int(rng, 1, 500))),
                      rng.choice((1.0, rng.uniform(0.5, 0.999))), rng.choice((0.0, rng.uniform(0.001, 0.3))),
                      rng.uniform(0.2, 2.0), rng.random() < 0.5)
    if kind == "append":
        tokens = rng.choice((1, 1, 1, log_int(rng, 2, 2000)))
        rows = log_int(rng, 1, 256 if tokens == 1 else max(1, 2000 // tokens))
        form, bits = rng.choice((("norm", 4), ("norm", 4), ("norm", 16), ("rope", 4), ("plain", 4)))
        return append(rows, tokens, tokens + log_int(rng, 1, 8000 - tokens), page, kv_heads, group,
                      rng.random() < 0.5, form, bits)
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


def work(case):
    """Each byte once: the visible positions' codes, queries in, outputs out, scores read and written; the appended
    vectors in, their codes out and in, and what these stand for out; the vectors in and out; the logits in."""
    c = case
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": 4 * n + c["rows"] * 28, "flops": 2 * n}
    if c["kind"] == "norm":
        n = c["rows"] * c["kv_heads"] * (c["group"] + 1) * c["head_dim"]
        return {"bytes": 4 * n + 4 * c["head_dim"], "flops": 9 * n}
    if c["kind"] == "attn":
        ns = lengths_of(c)
        heads, seen = c["kv_heads"] * c["group"], sum(ns)
        b = seen * 2 * c["kv_heads"] * VECTOR + 2 * c["rows"] * heads * HEAD_DIM * 2
        b += 4 * sum(pages_of(n, c["page"]) for n in ns) + 4 * c["rows"]
        if c["scored"]:
            b += 8 * seen * c["kv_heads"]
        return {"bytes": b, "flops": 4 * HEAD_DIM * heads * seen}
    n = c["rows"] * c["tokens"]
    heads = n * c["kv_heads"]
    b = 2 * heads * (256 + 2 * (VECTOR if c["bits"] == 4 else 256) + 256) + 8 * c["rows"]
    if c["form"] != "plain":
        b += 2 * heads * 256 * c["group"]
    if c["scored"]:
        b += 4 * heads
    return {"bytes": b, "flops": 9 * HEAD_DIM * heads * (c["group"] + 2)}


# ---- states ----

class State:
    """What the program holds: the pool, the rows' pages and lengths, scores, this step's vectors or logits."""


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


def packed(x):
    """Values [...][128] FP32 as vectors [...][80] of bytes."""
    x = x.view(*x.shape[:-1], 4, 32)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m = low.half()
    step = (high - low) / 15
    d = step.half()
    d = (d.view(torch.int16) - (d.float() > step).short()).view(torch.float16)  # cut off, not rounded
    code = torch.where(d > 0, (x - m.float()) / d.float(), torch.zeros_like(x))
    code = code.round().clamp(0, 15).to(torch.uint8).flatten(-2)
    dm = torch.cat([d, m], -1).flatten(-2).contiguous().view(torch.uint8)
    return torch.cat([code[..., 0::2] | code[..., 1::2] << 4, dm], -1)


def unpacked(b):
    """Vectors [...][80] of bytes as the FP32 values [...][128] that they stand for."""
    codes = b[..., :64]
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    dm = b[..., 64:].contiguous().view(torch.float16).float()
    d, m = dm[..., 0::2, None], dm[..., 1::2, None]
    return (codes.view(*codes.shape[:-1], 4, 32) * d + m).flatten(-2)


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


def norm_weight(g, n):
    return (1 + 0.2 * normal(g, n, dtype=torch.float32)).half()


def sampling_inputs(c, s, g):
    """Logits as a model's: most tokens in a broad heap, a few dozen candidates that stand out."""
    rows, vocab = c["rows"], c["vocab"]
    x = 2.2 * normal(g, rows, vocab, dtype=torch.float32)
    best = torch.randint(0, vocab, (rows, 60), generator=g, device="cuda")
    lift = 14 * torch.rand(rows, 60, generator=g, device="cuda") ** 2
    s.logits = x.scatter_add(1, best, lift + 2)
    u = torch.rand(rows, 5, generator=g, device="cuda")
    t = torch.full((rows,), c["temperature"], device="cuda")
    k = torch.full((rows,), c["top_k"], device="cuda", dtype=torch.int64)
    p, m = torch.full((rows,), c["top_p"], device="cuda"), torch.full((rows,), c["min_p"], device="cuda")
    if c["mixed"]:
        t = torch.where(u[:, 0] < 0.1, torch.zeros_like(t), t * (0.5 + u[:, 0]))
        k = torch.where(u[:, 1] < 0.3, torch.zeros_like(k), (k * 2 * u[:, 1]).long() + 1)
        p = torch.where(u[:, 2] < 0.3, torch.ones_like(p), 1 - (1 - p) * 2 * u[:, 2])
        m = torch.where(u[:, 3] < 0.5, torch.zeros_like(m), m * u[:, 3])
    # per row: temperature, top_p, top_k (a whole number), min_p
    s.params = torch.stack([t.view(torch.int32), p.view(torch.int32), k.int(), m.view(torch.int32)], 1).contiguous()
    s.uniform = torch.rand(rows, generator=g, device="cuda")
    s.tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    s.probs = torch.zeros(rows, device="cuda")


def inputs(c, seed):
    """A case's tensors, from the seed alone."""
    g, s = generator(seed), State()
    s.case = c
    if c["kind"] == "sample":
        sampling_inputs(c, s, g)
        return s
    heads = c["kv_heads"] * c["group"]
    if c["kind"] == "norm":
        dim = c["head_dim"]
        s.q, s.k = 2 * normal(g, c["rows"], heads, dim), 3 * normal(g, c["rows"], c["kv_heads"], dim)
        s.q_norm, s.k_norm = norm_weight(g, dim), norm_weight(g, dim)
        return s
    ns = lengths_of(c)
    s.width = pages_of(max(ns), c["page"])
    capacity = s.width * c["page"]
    s.lengths = torch.tensor(ns, device="cuda", dtype=torch.int64)
    if c["kind"] == "append":
        # what lies before the new tokens is a shared prefix: only the pages that are written are the rows' own
        first = [(n - c["tokens"]) // c["page"] for n in ns]
        mine, pages = scatter_pages(g, [n - f * c["page"] for n, f in zip(ns, first)], c["page"], s.width, 1)
        at = torch.arange(s.width, device="cuda")[None] - torch.tensor(first, device="cuda")[:, None]
        s.table = torch.where(at >= 0, torch.gather(mine, 1, at.clamp(min=0)), torch.zeros_like(mine))
        shape = (c["rows"], c["tokens"])
        s.q = normal(g, *shape, heads, HEAD_DIM)
        s.k, s.v = (normal(g, *shape, c["kv_heads"], HEAD_DIM) for _ in range(2))
        s.out, s.k_out, s.v_out = torch.empty_like(s.q), torch.empty_like(s.k), torch.empty_like(s.v)
        s.q_norm, s.k_norm = norm_weight(g, HEAD_DIM), norm_weight(g, HEAD_DIM)
        # a sequence that lost positions to an eviction stands further on than its length says
        gap = torch.randint(0, 100, (c["rows"],), generator=g, device="cuda")
        s.positions = s.lengths - c["tokens"] + gap
        s.most = max(ns) + 100
    else:
        s.table, pages = scatter_pages(g, ns, c["page"], s.width)
        s.q = normal(g, c["rows"], heads, HEAD_DIM)
        s.out = torch.empty_like(s.q)
    s.slots = pages * c["page"]
    if c.get("bits", 4) == 16:
        s.kc, s.vc = (normal(g, s.slots, c["kv_heads"], HEAD_DIM) for _ in range(2))
    else:
        s.kc, s.vc = (torch.empty(s.slots, c["kv_heads"], VECTOR, dtype=torch.uint8, device="cuda") for _ in range(2))
        for cache in (s.kc, s.vc):
            for part in cache.split(1 << 16):
                part.copy_(packed(normal(g, part.shape[0], c["kv_heads"], HEAD_DIM, dtype=torch.float32)))
    s.score = None
    if c["scored"]:
        # accumulated weights are far from even, and some positions were never attended to
        z = normal(g, c["rows"], c["kv_heads"], capacity, dtype=torch.float32)
        s.score = torch.where(z < -1.5, torch.zeros_like(z), (2 * z).exp())
    return s


def handle(t):
    from graph_horizon_amd import _ffi as F
    return F.GhBuf(t.data_ptr(), t.numel() * t.element_size(), 0, F.BUF_VIEW, 0, 0)


def paged(s):
    """The framework's handle of a paged cache."""
    from graph_horizon_amd import _ffi as F
    c = s.case
    scheme = F.KV_F16 if c.get("bits", 4) == 16 else F.KV_Q4
    kv = F.GhKv(handle(s.kc), handle(s.vc), scheme, 1, s.slots, c["kv_heads"], HEAD_DIM, HEAD_DIM)
    return F.GhKvPaged(kv, handle(s.table), handle(s.lengths), F.GhBuf() if s.score is None else handle(s.score),
                       c["page"], s.width, c["rows"])


def prepare(case, seed):
    s = inputs(case, seed)
    for name in ("table", "lengths", "positions"):  # 32-bit on the device, as the server keeps them
        if hasattr(s, name):
            setattr(s, name, getattr(s, name).to(torch.int32))
    if own:
        backend()
        from graph_horizon_amd import Yarn
        s.yarn = Yarn(**dict(YARN, rope_dim=case.get("head_dim", HEAD_DIM)))
        s.buf = {n: handle(t) for n, t in vars(s).items() if isinstance(t, torch.Tensor)}
        if hasattr(s, "table"):
            s.kv = paged(s)
    return s


# ---- one pass ----

def run(s):
    c = s.case
    if c["kind"] == "attn":
        (attn_own if own else attn_plain)(s)
        return {"out": s.out} if s.score is None else {"out": s.out, "score": s.score}
    if c["kind"] == "append":
        (append_own if own else append_plain)(s)
        got = {"k": s.k_out, "v": s.v_out}
        if c["form"] != "plain":
            got["q"] = s.out
        if s.score is not None:
            got["score"] = s.score
        return got
    if c["kind"] == "norm":
        (norm_own if own else norm_plain)(s)
        return {"q": s.q, "k": s.k}
    (sample_own if own else sample_plain)(s)
    return {"tokens": s.tokens, "probs": s.probs}


def attn_own(s):
    c = s.case
    backend().attention_decode_paged(s.buf["out"], s.buf["q"], s.kv, c["kv_heads"] * c["group"], c["length"], 0)


def append_own(s):
    """The append, and what the pool then holds for the new tokens."""
    c, b, hip = s.case, s.buf, backend()
    heads = c["kv_heads"] * c["group"]
    hip.begin()
    if c["form"] == "norm":
        hip.norm_rope_kv_write_paged(s.kv, b["out"], b["q"], b["k"], b["v"], heads, b["q_norm"], b["k_norm"], EPS,
                                     b["positions"], c["tokens"], s.most, s.yarn, 0)
    elif c["form"] == "rope":
        hip.rope_kv_write_paged(s.kv, b["out"], b["q"], b["k"], b["v"], heads, b["positions"], c["tokens"], s.most,
                                s.yarn, 0)
    else:
        hip.kv_write_paged(s.kv, b["k"], b["v"], c["tokens"], 0)
    hip.kv_read_paged(b["k_out"], b["v_out"], s.kv, c["tokens"], 0)
    hip.submit()


def norm_own(s):
    c, b = s.case, s.buf
    backend().norm_rope_batched(b["q"], b["k"], c["kv_heads"] * c["group"], c["kv_heads"], c["head_dim"], c["base"],
                                c["rows"], b["q_norm"], b["k_norm"], EPS, s.yarn)


def sample_own(s):
    c, b = s.case, s.buf
    backend().sample_rows(b["tokens"], b["probs"], b["logits"], c["rows"], c["vocab"], c["vocab"], b["params"],
                          b["uniform"])


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
    k = unpacked(s.kc[slots]).permute(0, 2, 3, 1).contiguous()  # [rows][kv heads][128][cap]
    q = s.q.view(rows, hk, g, HEAD_DIM).float()
    x = torch.matmul(q, k) * (1 / math.sqrt(HEAD_DIM))
    del k
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(seen.any(-1)[:, None, None, None], top, torch.zeros_like(top)))
    p = p / p.sum(-1, keepdim=True)
    p = torch.where(seen[:, None, None], p, torch.zeros_like(p))
    v = unpacked(s.vc[slots]).permute(0, 2, 1, 3).contiguous()
    v = v.masked_fill_(~seen[:, None, :, None], 0)
    s.out.copy_(torch.matmul(p, v).view(rows, hk * g, HEAD_DIM))
    if s.score is not None:
        s.score[:, :, :cap] += p.sum(2)


def corrections(dim):
    """The pairs between which YaRN goes over from the plain angle to the interpolated one."""
    y = YARN

    def corr(turns):
        return dim * math.log(y["original_context"] / (turns * 2 * math.pi)) / (2 * math.log(y["freq_base"]))

    return max(math.floor(corr(y["beta_fast"])), 0), min(math.ceil(corr(y["beta_slow"])), dim - 1)


def angles(pos, dim):
    """YaRN's angle of each pair at the positions. It is an FP32 number by the operators' definition, step by step,
    so that an appended key is the one that a prefill would have written; what follows from it is held in 64 bits."""
    pair = torch.arange(dim // 2, device="cuda")
    lo, hi = corrections(dim)
    ramp = 1 - ((pair.float() - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    turned = pos.float()[..., None] * (YARN["freq_base"] ** (-2 * pair.double() / dim)).float()
    return (turned * (1 / YARN["factor"]) * (1 - ramp) + turned * ramp).double()


def post_scale(pos):
    """Queries past the original context are scaled up."""
    return ((pos // YARN["original_context"]).double() + 1).log() * YARN["q_temperature_scale"] + 1


def normed(x, weight):
    """x [...][dim] over the root of its mean square, times the weight, in 32 bits."""
    x = x.float()
    return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.float()


def rotated(x, pos, query):
    """x [...][heads][dim] in FP32 with adjacent pairs turned by the angles at pos [...]."""
    t = angles(pos, x.shape[-1])[..., None, :]
    scale = post_scale(pos)[..., None, None] if query else 1
    cos, sin = (t.cos() * scale).float(), (t.sin() * scale).float()
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).view(x.shape)


def append_plain(s):
    c = s.case
    step = torch.arange(c["tokens"], device="cuda")[None]
    at = s.lengths.long()[:, None] - c["tokens"] + step
    slots = slots_of(s.table, c["page"], at)
    q, k, v = s.q.float(), s.k.float(), s.v.float()
    if c["form"] == "norm":
        q, k = normed(q, s.q_norm), normed(k, s.k_norm)
    if c["form"] != "plain":
        pos = s.positions.long()[:, None] + step
        s.out.copy_(rotated(q, pos, True))
        k = rotated(k, pos, False)
    if c["bits"] == 4:
        s.kc[slots], s.vc[slots] = packed(k), packed(v)
        s.k_out.copy_(unpacked(s.kc[slots]))
        s.v_out.copy_(unpacked(s.vc[slots]))
    else:
        s.kc[slots], s.vc[slots] = k.half(), v.half()
        s.k_out.copy_(s.kc[slots])
        s.v_out.copy_(s.vc[slots])
    if s.score is not None:
        row = torch.arange(c["rows"], device="cuda")[:, None].expand_as(at)
        s.score[row, :, at] = 0


def norm_plain(s):
    c = s.case
    pos = torch.arange(c["rows"], device="cuda") + c["base"]
    s.q.copy_(rotated(normed(s.q, s.q_norm), pos, True))
    s.k.copy_(rotated(normed(s.k, s.k_norm), pos, False))


def sample_plain(s):
    """Tokens in order of their logits (equal ones: the lowest first). Weights exp((logit - largest) / temperature):
    the first top_k of them, of those the fewest whose weights reach top_p of the sum, of those the ones that are at
    least min_p of the largest; then the first at which the running sum passes uniform times the sum. In 64 bits:
    sums over a vocabulary, and values next to a border."""
    c = s.case
    t, p, m = (s.params[:, i].contiguous().view(torch.float32).double()[:, None] for i in (0, 1, 3))
    k = s.params[:, 2:3]
    x, order = torch.sort(s.logits, dim=-1, descending=True, stable=True)
    rank = torch.arange(c["vocab"], device="cuda")[None]
    greedy = t <= 0
    k = torch.where(greedy, torch.ones_like(k), torch.where(k > 0, k, torch.full_like(k, c["vocab"])))
    w = torch.exp((x.double() - x[:, :1].double()) / torch.where(greedy, torch.ones_like(t), t))
    w = torch.where(rank < k, w, torch.zeros_like(w))
    before = torch.cumsum(w, -1) - w
    keep = (before < p * w.sum(-1, keepdim=True)) | (p >= 1)
    keep &= w >= m
    keep[:, 0] = True
    w = torch.where(keep, w, torch.zeros_like(w))
    upto = torch.cumsum(w, -1)
    total = upto[:, -1:]
    past = (upto > s.uniform.double()[:, None] * total) & (w > 0)
    at = torch.argmax(past.to(torch.uint8), -1, keepdim=True)
    s.tokens.copy_(torch.gather(order, 1, at)[:, 0])
    s.probs.copy_((torch.gather(w, 1, at) / total)[:, 0])


# ---- the same in 64 bits ----

def exact(case, seed):
    s = inputs(case, seed)
    return {"attn": exact_attn, "append": exact_append, "norm": exact_norm, "sample": exact_sample}[case["kind"]](s)


def cells(s, r, n):
    """The slots of row r's first n positions, in order."""
    p = s.case["page"]
    pages = s.table[r, :pages_of(n, p)].tolist()
    return torch.cat([torch.arange(x * p, x * p + p, device="cuda") for x in pages])[:n]


def exact_values(b):
    """Bytes [n][80] as 64-bit values: dim i has half a byte of codes and a pair of FP16 numbers."""
    i = torch.arange(HEAD_DIM, device="cuda")
    code = (b[:, i // 2].long() >> (4 * (i % 2))) & 15
    at = 64 + 4 * (i // 32)

    def half(at):
        bits = b[:, at].long() | b[:, at + 1].long() << 8
        e, f = bits >> 10 & 31, (bits & 1023).double()
        size = torch.where(e > 0, (1024 + f) * torch.exp2(e.double() - 25), f * 2.0 ** -24)
        return torch.where(bits >> 15 > 0, -size, size)

    return half(at + 2) + half(at) * code


def exact_attn(s):
    c = s.case
    out = torch.zeros(c["rows"], c["kv_heads"], c["group"], HEAD_DIM, dtype=torch.float64, device="cuda")
    score = None if s.score is None else s.score.double()
    for r, n in enumerate(lengths_of(c)):
        if n == 0:
            continue
        at = cells(s, r, n)
        for h in range(c["kv_heads"]):
            k, v = exact_values(s.kc[at, h]), exact_values(s.vc[at, h])
            q = s.q[r, h * c["group"]:(h + 1) * c["group"]].double()
            w = torch.softmax(q @ k.t() / math.sqrt(HEAD_DIM), -1)
            out[r, h] = w @ v
            if score is not None:
                score[r, h, :n] += w.sum(0)
    out = out.view(c["rows"], -1, HEAD_DIM)
    return {"out": out} if score is None else {"out": out, "score": score}


def exact_turn(x, positions, query):
    """x [n][heads][dim] in 64 bits, rotated at n positions. The angles are the FP32 ones of the definition."""
    f, y, dim = np.float32, YARN, x.shape[-1]
    pair = np.arange(dim // 2)
    freq = np.power(y["freq_base"], -2.0 * pair / dim).astype(f)
    lo, hi = corrections(dim)
    ramp = f(1) - np.clip((pair.astype(f) - f(lo)) / f(max(hi - lo, 0.001)), f(0), f(1))
    far = np.asarray(positions, f)[:, None] * freq
    theta = (f(1 / y["factor"]) * far) * (f(1) - ramp) + far * ramp
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], dim // 2, 2).contiguous())
    turn = torch.from_numpy(np.exp(1j * theta.astype(np.float64))).cuda()
    if query:
        up = 1 + y["q_temperature_scale"] * np.log1p(np.asarray(positions) // y["original_context"])
        turn = turn * torch.from_numpy(up).cuda()[:, None]
    return torch.view_as_real(z * turn[:, None]).reshape(x.shape)


def exact_norm_of(x, weight):
    x = x.double()
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()


def exact_codes(x):
    """What [n][heads][128] values are held as, from the definition in 64 bits."""
    x = x.view(-1, 32)
    low = x.min(1).values
    d = (x.max(1).values - low) / 15
    m = low.half().double()
    unit = torch.exp2(torch.frexp(d).exponent.clamp(min=-13).double() - 11)  # of the FP16 numbers around d
    d = torch.floor(d / unit) * unit
    code = torch.round((x - m[:, None]) / torch.where(d == 0, torch.ones_like(d), d)[:, None])
    return m[:, None] + d[:, None] * torch.clamp(code, 0, 15)


def exact_append(s):
    c = s.case
    rows, tokens = c["rows"], c["tokens"]
    n = rows * tokens
    at = [p + t for p in s.positions.tolist() for t in range(tokens)]
    q, k, v = (x.double().view(n, -1, HEAD_DIM) for x in (s.q, s.k, s.v))
    if c["form"] == "norm":
        q, k = exact_norm_of(q, s.q_norm), exact_norm_of(k, s.k_norm)
    if c["form"] != "plain":
        q, k = exact_turn(q, at, True), exact_turn(k, at, False)
    if c["bits"] == 4:
        k, v = exact_codes(k), exact_codes(v)
    got = {"k": k.view(s.k.shape), "v": v.view(s.v.shape)}
    if c["form"] != "plain":
        got["q"] = q.view(s.q.shape)
    if s.score is not None:
        got["score"] = s.score.double()
        for r, length in enumerate(lengths_of(c)):
            got["score"][r, :, length - tokens:length] = 0
    return got


def exact_norm(s):
    c = s.case
    at = range(c["base"], c["base"] + c["rows"])
    return {"q": exact_turn(exact_norm_of(s.q, s.q_norm), at, True),
            "k": exact_turn(exact_norm_of(s.k, s.k_norm), at, False)}


def exact_sample(s):
    c = s.case
    logits, uniform = s.logits.double().cpu().numpy(), s.uniform.double().cpu().numpy()
    params = s.params.cpu().numpy()
    tokens, probs = [], []
    for r in range(c["rows"]):
        t, p, m = (float(params[r, i:i + 1].view(np.float32)[0]) for i in (0, 1, 3))
        k = int(params[r, 2])
        order = np.lexsort((np.arange(c["vocab"]), -logits[r]))
        order = order[:1] if t <= 0 else order[:k] if k else order
        w = np.exp((logits[r, order] - logits[r, order[0]]) / (t if t > 0 else 1))
        if p < 1:
            w = w[:np.searchsorted(np.cumsum(w), p * w.sum()) + 1]
        w = w[:max(1, int((w >= m).sum()))]
        upto = np.cumsum(w)
        i = min(int(np.searchsorted(upto, uniform[r] * upto[-1], side="right")), len(w) - 1)
        tokens.append(int(order[i]))
        probs.append(w[i] / upto[-1])
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "probs": torch.tensor(probs, dtype=torch.float64)}
