"""The operators of a served step over a shared prefix, as cases to time: keys and values appended to the paged cache (with norms and rotation on the
way), attention of a batch over a prefix that its rows share and over each row's own tokens, and a token drawn from each row of logits.

`run` computes a case in plain torch where `own` is false, and through `tlaloc_b200.ops` where it is true.
"""
import math

import numpy as np
import torch

own = False
DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f8": torch.float8_e4m3fn}
BYTES = {"f32": 4, "bf16": 2, "f8": 1}


def listed() -> list:
    return [
        # one sequence decodes: latency
        dict(name="append one token", kind="append", tokens=1, heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, norm=True, x="f32", pool="bf16", query="bf16", block=16),
        # a full decode batch on an 8-bit cache
        dict(name="append 128 sequences", kind="append", tokens=128, heads=64, kv_heads=8, dim=128, rot=128, interleaved=False, norm=True, x="f32", pool="f8", query="f32", block=16),
        # a prompt's tokens, half of each head rotated in pairs
        dict(name="append a prompt", kind="append", tokens=8192, heads=32, kv_heads=8, dim=128, rot=64, interleaved=True, norm=True, x="bf16", pool="bf16", query="bf16", block=64),
        # odd sizes, no norms, f32 throughout
        dict(name="append odd sizes", kind="append", tokens=1777, heads=20, kv_heads=5, dim=80, rot=48, interleaved=False, norm=False, x="f32", pool="f32", query="f32", block=24),
        # two continuations of a short prompt: latency
        dict(name="prefix of two rows", kind="prefix", groups=1, rows=2, prefix=500, own=64, heads=32, kv_heads=8, dim=128, block=16, pool="bf16", query="bf16", out="bf16"),
        # a system prompt before 64 conversations, as the decode step has its types
        dict(name="prefix of 64 rows", kind="prefix", groups=1, rows=64, prefix=8192, own=1024, heads=32, kv_heads=8, dim=128, block=16, pool="bf16", query="f32", out="bf16"),
        # a long document before a full batch
        dict(name="long prefix of 128 rows", kind="prefix", groups=1, rows=128, prefix=32768, own=512, heads=64, kv_heads=8, dim=128, block=16, pool="bf16", query="bf16", out="bf16"),
        # several samples of each of 24 prompts
        dict(name="prefixes of 24 prompts", kind="prefix", groups=24, rows=96, prefix=3000, own=300, heads=16, kv_heads=4, dim=64, block=32, pool="bf16", query="bf16", out="f32"),
        # an 8-bit cache
        dict(name="8-bit prefix of 40 rows", kind="prefix", groups=1, rows=40, prefix=10000, own=700, heads=32, kv_heads=8, dim=128, block=16, pool="f8", query="bf16", out="bf16"),
        # one request
        dict(name="draw one token", kind="sample", rows=1, vocab=128256, settings="all", logits="f32"),
        # a batch of requests with settings of their own: greedy ones, unfiltered ones, any of the filters
        dict(name="draw 128 tokens", kind="sample", rows=128, vocab=128256, settings="mixed", logits="f32"),
        # temperature alone: the whole vocabulary stays in
        dict(name="draw 512 unfiltered", kind="sample", rows=512, vocab=32768, settings="temperature", logits="bf16"),
    ]


def _cost(case) -> float:
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number from lo to hi, its logarithm uniform."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """One more case of these ranges; one that would cost more than the largest listed one of its kind is drawn again, and one over a 32-bit cache (which
    no configuration here has for more than small models) beyond 20 GFLOP."""
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("append", "prefix", "sample")}
    while True:
        c = _drawn(rng)
        if _cost(c) <= most[c["kind"]] and not (c["kind"] == "prefix" and c["pool"] == "f32" and work(c)["flops"] > 2e10):
            return c


def _drawn(rng) -> dict:
    kind = rng.choice(["append", "prefix", "prefix", "sample"])
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (8, 1), (16, 16), (20, 5), (24, 8), (4, 2), (16, 4)])
    if kind == "append":
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256])
        return dict(kind=kind, tokens=_spread(rng, 1, 8192), heads=heads, kv_heads=kv_heads, dim=dim, rot=rng.choice([dim, dim, dim // 2, dim // 4]),
                    interleaved=rng.random() < 0.4, norm=rng.random() < 0.7, x=rng.choice(["f32", "bf16"]), pool=rng.choice(["bf16", "bf16", "f8", "f32"]),
                    query=rng.choice(["f32", "bf16"]), block=rng.choice([16, 16, 24, 64]))
    if kind == "prefix":
        rows = _spread(rng, 1, 128)
        return dict(kind=kind, groups=rng.choice([1, 1, min(rows, 4), min(rows, 16)]), rows=rows, prefix=_spread(rng, 1, 32768), own=_spread(rng, 1, 1024), heads=heads,
                    kv_heads=kv_heads, dim=rng.choice([64, 64, 80, 128, 128, 128, 128, 256]), block=rng.choice([16, 16, 16, 24, 32, 64]),
                    pool=rng.choice(["bf16", "bf16", "bf16", "f8", "f32"]), query=rng.choice(["f32", "bf16"]), out=rng.choice(["f32", "bf16"]))
    return dict(kind=kind, rows=_spread(rng, 1, 512), vocab=rng.choice([1000, 1024, 4099, 32000, 32768, 50257, 100352, 128256, 151937, 262144]),
                settings=rng.choice(["all", "mixed", "mixed", "temperature", "top_k", "top_p", "min_p"]), logits=rng.choice(["f32", "f32", "bf16"]))


# ------------------------------------------------------------------------------------------------ sizes that follow from a case

def _group_rows(case) -> np.ndarray:
    """First rows of the groups, and the end: the rows shared out unevenly, one at least to each."""
    g, rows = case["groups"], case["rows"]
    weight = 1.0 + np.arange(g) % 3
    at = np.floor(np.cumsum(weight) / weight.sum() * (rows - g) + 1e-9).astype(np.int64) + np.arange(1, g + 1)
    return np.concatenate([[0], at]).astype(np.int32)


def _prefix_lengths(case) -> np.ndarray:
    """Lengths of the prefixes: the first has the case's, the others less."""
    g = case["groups"]
    return np.maximum(1, np.round(np.linspace(case["prefix"], max(1, case["prefix"] // 16), g))).astype(np.int32)


def _own_lengths(case) -> np.ndarray:
    """Own tokens of the rows: from one to the case's."""
    return np.round(np.linspace(1, case["own"], case["rows"])).astype(np.int32)[::-1].copy() if case["rows"] > 1 else np.array([case["own"]], np.int32)


def work(case) -> dict:
    """Each input read once, each output written once; two products a (row, head, key)."""
    if case["kind"] == "append":
        t, d = case["tokens"], case["dim"]
        q, kv = t * case["heads"] * d, t * 2 * case["kv_heads"] * d
        moved = (q + kv) * BYTES[case["x"]] + q * BYTES[case["query"]] + kv * BYTES[case["pool"]]
        return {"bytes": moved + t * (8 + case["rot"] * 4) + (8 * d if case["norm"] else 0), "flops": 8 * (q + kv // 2)}
    if case["kind"] == "prefix":
        starts, lens, tail = _group_rows(case), _prefix_lengths(case), _own_lengths(case)
        seen = int(np.sum(np.diff(starts).astype(np.int64) * lens)) + int(tail.sum())
        kept = int(lens.sum()) + int(tail.sum())
        rows, h, d = case["rows"], case["heads"], case["dim"]
        pages = sum(-(-int(n) // case["block"]) for n in (*lens, *tail))
        return {"bytes": kept * 2 * case["kv_heads"] * d * BYTES[case["pool"]] + rows * h * d * (BYTES[case["query"]] + BYTES[case["out"]]) + 4 * pages + 4 * rows,
                "flops": 4 * seen * h * d}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * BYTES[case["logits"]] + case["rows"] * 24, "flops": 4 * n}


# ------------------------------------------------------------------------------------------------ what a program has in hand

def prepare(case, seed) -> dict:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    rng = np.random.RandomState(int(seed) % (1 << 31))
    return {"append": _prepare_append, "prefix": _prepare_prefix, "sample": _prepare_sample}[case["kind"]](case, g, rng)


def _normal(g, *shape):
    return torch.randn(shape, device=DEVICE, generator=g)


def _prepare_append(case, g, rng) -> dict:
    t, h, hk, d, block = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["block"]
    x = (_normal(g, t, (h + 2 * hk) * d) * (0.5 + torch.rand((t, 1), device=DEVICE, generator=g))).to(TYPES[case["x"]])  # one projection's rows: [q | k | v]
    pages = -(-t // block) + 8
    where = rng.permutation(pages * block)[:t] if t < 512 else (rng.permutation(pages).astype(np.int64)[:, None] * block + np.arange(block)).reshape(-1)[:t]  # a prompt's pages in any order
    first = int(rng.randint(0, 4000))
    positions = first + np.arange(t) if t >= 512 else rng.randint(0, 12000, t)
    # angles of positions stretched by four, as a context longer than the trained one has them; computed in 64 bits
    freq = 10000.0 ** (-2.0 * np.arange(case["rot"] // 2) / max(case["rot"], 1)) / 4.0
    angle = np.arange(12288)[:, None] * freq[None, :]
    put = lambda a, kind: torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE).to(kind)  # noqa: E731
    pool = lambda: torch.zeros((pages, block, hk, d), device=DEVICE).to(TYPES[case["pool"]])  # noqa: E731
    return dict(case=case, q=x[:, :h * d].unflatten(1, (h, d)), k=x[:, h * d:(h + hk) * d].unflatten(1, (hk, d)), v=x[:, (h + hk) * d:].unflatten(1, (hk, d)),
                q_gain=1 + 0.1 * _normal(g, d) if case["norm"] else None, k_gain=1 + 0.1 * _normal(g, d) if case["norm"] else None, eps=1e-6,
                positions=put(positions, torch.int32), cos=put(np.cos(angle), torch.float32), sin=put(np.sin(angle), torch.float32),
                slots=put(where, torch.int32), key_cache=pool(), value_cache=pool())


def _prepare_prefix(case, g, rng) -> dict:
    h, hk, d, block, rows = case["heads"], case["kv_heads"], case["dim"], case["block"], case["rows"]
    starts, lens, tail = _group_rows(case), _prefix_lengths(case), _own_lengths(case)
    counts = [-(-int(n) // block) for n in (*lens, *tail)]
    order = rng.permutation(sum(counts) + 1).astype(np.int32)
    prefix_tables = np.zeros((len(lens), max(counts[:len(lens)])), np.int32)
    tables = np.zeros((rows, -(-case["own"] // block)), np.int32)
    at = 0
    for i, n in enumerate(counts):
        (prefix_tables[i] if i < len(lens) else tables[i - len(lens)])[:n] = order[at:at + n]
        at += n
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEVICE)  # noqa: E731
    pool = lambda: _normal(g, len(order), block, hk, d).to(TYPES[case["pool"]])  # noqa: E731
    return dict(case=case, query=(2.0 * _normal(g, rows, h, d)).to(TYPES[case["query"]]), key_cache=pool(), value_cache=pool(), prefix_tables=put(prefix_tables),
                prefix_lens=put(lens), row_starts=put(starts), tables=put(tables), lens=put(tail), scale=d ** -0.5,
                host=dict(starts=starts.tolist(), lens=lens.tolist()))


def _settings(case, rng):
    """(temperature, top_k, top_p, min_p) of the rows."""
    rows, kind = case["rows"], case["settings"]
    temperature = rng.uniform(0.6, 1.3, rows)
    top_k, top_p, min_p = np.zeros(rows, np.int64), np.ones(rows), np.zeros(rows)
    some = lambda share: rng.uniform(size=rows) < share  # noqa: E731
    if kind in ("all", "top_k", "mixed"):
        top_k = np.where(some(1.0 if kind != "mixed" else 0.4), rng.choice([1, 8, 40, 50, 64, 200, 1000], rows), 0)
    if kind in ("all", "top_p", "mixed"):
        top_p = np.where(some(1.0 if kind != "mixed" else 0.5), rng.choice([0.1, 0.5, 0.8, 0.9, 0.95, 0.99], rows), 1.0)
    if kind in ("all", "min_p", "mixed"):
        min_p = np.where(some(1.0 if kind != "mixed" else 0.3), rng.choice([0.02, 0.05, 0.1], rows), 0.0)
    if kind == "mixed":
        temperature = np.where(some(0.15), 0.0, temperature)  # greedy requests beside the others
    return temperature, top_k, top_p, min_p


def _prepare_sample(case, g, rng) -> dict:
    rows, n = case["rows"], case["vocab"]
    spread = torch.rand((rows, 1), device=DEVICE, generator=g) * 2.5 + 1.0
    logits = _normal(g, rows, n) * spread
    sure = torch.rand((rows, 1), device=DEVICE, generator=g) < 0.5  # rows that know what comes: a few tokens far above the rest
    logits += torch.where(sure & (torch.rand((rows, n), device=DEVICE, generator=g) < 8.0 / n), 12.0, 0.0)
    masked = torch.rand((rows, 1), device=DEVICE, generator=g) < 0.15  # rows under a grammar: most tokens are out
    logits.masked_fill_(masked & (torch.rand((rows, n), device=DEVICE, generator=g) < 0.9), -math.inf)
    temperature, top_k, top_p, min_p = _settings(case, rng)
    put = lambda a, kind: torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE).to(kind)  # noqa: E731
    return dict(case=case, logits=logits.to(TYPES[case["logits"]]), uniforms=torch.rand((rows,), device=DEVICE, generator=g), temperature=put(temperature, torch.float32),
                top_k=put(top_k, torch.int32), top_p=put(top_p, torch.float32), min_p=put(min_p, torch.float32))


# ------------------------------------------------------------------------------------------------ a pass

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "prefix": _own_prefix, "sample": _own_sample}[kind](state)
    return {"append": _plain_append, "prefix": _plain_prefix, "sample": _plain_sample}[kind](state)


def _own_append(s):
    from tlaloc_b200 import ops

    q = ops.norm_rope_kv_write(s["q"], s["k"], s["v"], s["positions"], s["cos"], s["sin"], s["slots"], s["key_cache"], s["value_cache"], q_gain=s["q_gain"],
                               k_gain=s["k_gain"], eps=s["eps"], interleaved=s["case"]["interleaved"], q_dtype=TYPES[s["case"]["query"]])
    return {"q": q, "keys": s["key_cache"], "values": s["value_cache"]}


def _own_prefix(s):
    from tlaloc_b200 import ops

    if "scratch" not in s:  # a program keeps the workspace of its step
        s["scratch"] = ops.shared_prefix_scratch(s["query"], s["key_cache"], s["prefix_tables"], s["tables"])
    return ops.shared_prefix_attention(s["query"], s["key_cache"], s["value_cache"], s["prefix_tables"], s["prefix_lens"], s["row_starts"], s["tables"], s["lens"],
                                       scale=s["scale"], out_dtype=TYPES[s["case"]["out"]], scratch=s["scratch"])


def _own_sample(s):
    from tlaloc_b200 import ops

    return ops.sample(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


def _plain_rotate(x, gain, s, cos, sin):
    """Norm over each head, then the rotation of its first channels, in 32 bits."""
    x = x.float()
    if gain is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * gain
    half = cos.shape[-1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if s["case"]["interleaved"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _narrow(x, kind):
    """Rounded to `kind`; 8 bits hold what lies past their largest value as that value."""
    return x.clamp(-448.0, 448.0).to(kind) if kind == torch.float8_e4m3fn else x.to(kind)


def _plain_append(s):
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q, k = _plain_rotate(s["q"], s["q_gain"], s, cos, sin), _plain_rotate(s["k"], s["k_gain"], s, cos, sin)
    slots, kind = s["slots"].long(), TYPES[s["case"]["pool"]]
    for cache, rows in ((s["key_cache"], k), (s["value_cache"], s["v"].float())):
        flat, rows = cache.view(-1, *cache.shape[2:]), _narrow(rows, kind)
        if kind == torch.float8_e4m3fn:  # indexing has no 8-bit form: the bytes
            flat, rows = flat.view(torch.uint8), rows.view(torch.uint8)
        flat[slots] = rows
    return {"q": _narrow(q, TYPES[s["case"]["query"]]), "keys": s["key_cache"], "values": s["value_cache"]}


def _pages(cache, tables):
    """The rows of the pages that tables [.., n] name: f32 [.., n * block, Hkv, D]."""
    if cache.dtype == torch.float8_e4m3fn:
        rows = cache.view(torch.uint8)[tables.long()].view(torch.float8_e4m3fn)
    else:
        rows = cache[tables.long()]
    return rows.float().flatten(-4, -3)


def _plain_prefix(s):
    q = s["query"].float()
    rows, h, d = q.shape
    hk, block = s["case"]["kv_heads"], s["case"]["block"]
    qg = q.view(rows, hk, h // hk, d)
    # own tokens: every row's pages, masked past its length
    k, v = _pages(s["key_cache"], s["tables"]), _pages(s["value_cache"], s["tables"])
    own_scores = torch.einsum("rkgd,rlkd->rkgl", qg, k) * s["scale"]
    own_scores.masked_fill_(torch.arange(k.shape[1], device=q.device) >= s["lens"][:, None, None, None], -math.inf)
    top = own_scores.amax(-1)
    p = torch.exp(own_scores - top[..., None])
    total, acc = p.sum(-1), torch.einsum("rkgl,rlkd->rkgd", p, v)
    out = torch.empty_like(acc)
    for i, length in enumerate(s["host"]["lens"]):
        lo, hi = s["host"]["starts"][i], s["host"]["starts"][i + 1]
        table = s["prefix_tables"][i, :-(-length // block)]
        k, v = _pages(s["key_cache"], table)[:length], _pages(s["value_cache"], table)[:length]
        flat = qg[lo:hi].transpose(0, 1).reshape(hk, -1, d)  # the rows and heads that read one key/value head, in one product
        scores = (flat @ k.permute(1, 2, 0)) * s["scale"]
        first = scores.amax(-1)
        both = torch.maximum(first, top[lo:hi].transpose(0, 1).reshape(hk, -1))
        p = torch.exp(scores - both[..., None])
        back = lambda x: x.view(hk, hi - lo, h // hk, *x.shape[2:]).transpose(0, 1)  # noqa: E731
        weight = torch.exp(top[lo:hi] - back(both))
        denominator = back(p.sum(-1)) + weight * total[lo:hi]
        out[lo:hi] = (back(p @ v.transpose(0, 1)) + weight[..., None] * acc[lo:hi]) / denominator[..., None]
    return out.view(rows, h, d).to(TYPES[s["case"]["out"]])


def _plain_sample(s):
    x = s["logits"].double()  # 64 bits: a draw falls next to a border of long sums
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    w = torch.exp((x - x.amax(1, keepdim=True)) / t)
    n = x.shape[1]
    order = torch.argsort(x, dim=1, descending=True, stable=True)
    ranked = w.gather(1, order)
    rank = torch.arange(n, device=x.device)[None]
    k = torch.where(s["top_k"] > 0, s["top_k"], n).long()[:, None]
    of_k = torch.where(rank < k, ranked, 0.0)
    sums = torch.cumsum(of_k, 1)
    before = torch.cat([torch.zeros_like(sums[:, :1]), sums[:, :-1]], 1)
    p = s["top_p"].double()[:, None]
    keep = (rank < k) & ((before < p * sums[:, -1:]) | (p >= 1) | (rank == 0)) & (ranked >= s["min_p"].double()[:, None])
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ranked, 0.0))
    sums = torch.cumsum(kept, 1)
    token = (sums <= s["uniforms"].double()[:, None] * sums[:, -1:]).sum(1)
    last = torch.where(kept > 0, rank, 0).amax(1)
    return torch.where(greedy, order[:, 0], torch.minimum(token, last)).to(torch.int32)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "prefix": _exact_prefix, "sample": _exact_sample}[case["kind"]](s)


def _exact_append(s):
    case = s["case"]
    rot, half = case["rot"], case["rot"] // 2
    c, sn = (s[name].double()[s["positions"].long()].unsqueeze(1) for name in ("cos", "sin"))
    # channel j of the result is x[j] * cos[f(j)] + sign(j) * x[partner(j)] * sin[f(j)]
    j = torch.arange(rot, device=DEVICE)
    partner, f, sign = (j ^ 1, j // 2, 2.0 * (j % 2) - 1) if case["interleaved"] else ((j + half) % max(rot, 1), j % max(half, 1), torch.where(j < half, -1.0, 1.0))

    def turned(x, gain):
        y = x.double()
        if gain is not None:
            y = y / torch.sqrt(y.pow(2).mean(2, keepdim=True) + s["eps"]) * gain.double()
        z = y.clone()
        z[..., :rot] = y[..., :rot] * c[..., f] + y[..., partner] * sn[..., f] * sign.double()
        return z

    def stored(rows):
        block = torch.zeros((s["key_cache"].shape[0] * case["block"], case["kv_heads"], case["dim"]), dtype=torch.float64, device=DEVICE)
        block[s["slots"].long()] = rows.clamp(-448, 448) if case["pool"] == "f8" else rows
        return block.view(s["key_cache"].shape)

    return {"q": turned(s["q"], s["q_gain"]), "keys": stored(turned(s["k"], s["k_gain"])), "values": stored(s["v"].double())}


def _exact_prefix(s):
    case = s["case"]
    rows, h, d = s["query"].shape
    per, block = h // case["kv_heads"], case["block"]
    out = torch.empty((rows, h, d), dtype=torch.float64, device=DEVICE)

    def gathered(cache, table, length, head):
        pos = torch.arange(length, device=DEVICE)
        return cache.view(torch.uint8 if case["pool"] == "f8" else cache.dtype)[table.long()[pos // block], pos % block, head].view(cache.dtype).double()

    lens = s["lens"].tolist()
    for i, length in enumerate(s["host"]["lens"]):
        lo, hi = s["host"]["starts"][i], s["host"]["starts"][i + 1]
        for kv in range(case["kv_heads"]):
            k, v = (gathered(s[c], s["prefix_tables"][i], length, kv) for c in ("key_cache", "value_cache"))
            q = s["query"][lo:hi, kv * per:(kv + 1) * per].double()
            scores = torch.einsum("rhd,ld->rhl", q, k) * s["scale"]
            parts = [(scores, v)]
            most = max(lens[lo:hi])
            kt = torch.zeros((hi - lo, most, d), dtype=torch.float64, device=DEVICE)
            vt = torch.zeros_like(kt)
            for r in range(lo, hi):
                kt[r - lo, :lens[r]], vt[r - lo, :lens[r]] = (gathered(s[c], s["tables"][r], lens[r], kv) for c in ("key_cache", "value_cache"))
            tail = torch.einsum("rhd,rld->rhl", q, kt) * s["scale"]
            tail[torch.arange(most, device=DEVICE)[None, None].expand_as(tail) >= s["lens"][lo:hi, None, None]] = -math.inf
            weights = torch.softmax(torch.cat([scores, tail], -1), -1)
            out[lo:hi, kv * per:(kv + 1) * per] = torch.einsum("rhl,ld->rhd", weights[..., :length], v) + torch.einsum("rhl,rld->rhd", weights[..., length:], vt)
    return out


def _exact_sample(s):
    logits, u = s["logits"].double().cpu().numpy(), s["uniforms"].double().cpu().numpy()
    settings = [s[name].double().cpu().numpy() for name in ("temperature", "top_k", "top_p", "min_p")]
    out = np.zeros((len(u),), np.int32)
    for r, x in enumerate(logits):
        t, k, p, m = (float(a[r]) for a in settings)
        if t <= 0:
            out[r] = int(np.argmax(x))
            continue
        w = np.exp((x - x.max()) / t)
        ranked = np.lexsort((np.arange(len(x)), -x))
        if k > 0:
            ranked = ranked[:int(k)]
        if p < 1:
            sums = np.cumsum(w[ranked])
            ranked = ranked[:1 + int(np.searchsorted(sums[:-1], p * sums[-1], side="left"))]
        ranked = np.sort(ranked[w[ranked] >= m])
        sums = np.cumsum(w[ranked])
        out[r] = ranked[min(int(np.searchsorted(sums, u[r] * sums[-1], side="right")), len(ranked) - 1)]
    return torch.from_numpy(out)
