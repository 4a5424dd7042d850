"""The serving operators of multi-sequence decode, as cases to measure.

Four operators that a decode step of many requests runs one after the other
(pyrite_b200.kernels.paged and pyrite_b200.kernels.sampling):

* ``tables``: block tables and slot maps from the requests' lengths;
* ``append``: QK-norm, RoPE and the new keys and values into their page slots;
* ``attend``: attention over a prefix that all requests share and over each
  request's own pages;
* ``sample``: temperature, top-k, top-p and min-p sampling from given random
  numbers.

``run`` computes a case either in plain torch operations (``own`` false) or by
the framework's calls (``own`` true); ``exact`` computes it in 64 bits from the
definition.
"""
import math
import random

import numpy as np
import torch

own = False

HEAD = 128
EPS = 1e-6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ITEM = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 16 requests (the batch decoder's default batch): a token each, some already finished
        {"name": "tables_step16", "op": "tables", "requests": 16, "page": 16, "width": 32, "held": 500, "new": 1,
         "padded": True},
        # 128 prompts admitted at once, up to 1024 tokens each, some continuing a partly filled page
        {"name": "tables_admit128", "op": "tables", "requests": 128, "page": 16, "width": 128, "held": 900,
         "new": 1024, "padded": False},
        # one decode step of 16 requests: 32 query and 8 key heads, no QK norm, 16-bit cache
        {"name": "append_step16", "op": "append", "rows": 16, "heads": 32, "kv_heads": 8, "norm": False, "page": 16,
         "dtype": "f16"},
        # a block of prompt positions of a model with QK norm, far into its context
        {"name": "append_block1537", "op": "append", "rows": 1537, "heads": 32, "kv_heads": 4, "norm": True,
         "page": 64, "dtype": "bf16"},
        # one request alone, a short context, the exact cache: latency
        {"name": "attend_one_f32", "op": "attend", "rows": 1, "heads": 16, "kv_heads": 8, "prefix": 0, "own": 97,
         "page": 16, "dtype": "f32"},
        # 16 requests behind a system prompt of 1000 tokens, the exact cache
        {"name": "attend_b16_f32", "op": "attend", "rows": 16, "heads": 16, "kv_heads": 8, "prefix": 1000, "own": 512,
         "page": 16, "dtype": "f32"},
        # 16 requests behind a long shared document, group of 8 heads, 16-bit cache
        {"name": "attend_b16_f16", "op": "attend", "rows": 16, "heads": 32, "kv_heads": 4, "prefix": 4096, "own": 500,
         "page": 16, "dtype": "f16"},
        # 64 requests behind a long shared document, group of 16 heads
        {"name": "attend_b64_bf16", "op": "attend", "rows": 64, "heads": 64, "kv_heads": 4, "prefix": 8191,
         "own": 1024, "page": 64, "dtype": "bf16"},
        # 24 requests that share nothing, long and of very different lengths
        {"name": "attend_long_f16", "op": "attend", "rows": 24, "heads": 32, "kv_heads": 8, "prefix": 0,
         "own": 16000, "page": 32, "dtype": "f16"},
        # one request's next token with the usual chat settings
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 151936, "mode": "chat"},
        # 16 requests, each with settings of its own, greedy and constrained ones among them
        {"name": "sample_b16_mixed", "op": "sample", "rows": 16, "vocab": 128256, "mode": "mixed"},
        # 128 requests by temperature and top-p over the whole vocabulary
        {"name": "sample_b128_open", "op": "sample", "rows": 128, "vocab": 151936, "mode": "open"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attend", "attend", "sample", "sample"])
    if op == "tables":
        requests, page = _log_int(rng, 1, 200), rng.choice([16, 32, 64, 128])
        padded = rng.random() < 0.5
        new = _log_int(rng, 1, 8) if padded else _log_int(rng, 1, 600)
        held = _log_int(rng, 1, 2000)
        return {"op": op, "requests": requests, "page": page, "width": (held + new + page - 1) // page + 1,
                "held": held, "new": new, "padded": padded}
    if op == "append":
        heads, kv_heads = rng.choice([(16, 8), (32, 8), (32, 4), (64, 4), (8, 8), (12, 3)])
        return {"op": op, "rows": _log_int(rng, 1, 1500), "heads": heads, "kv_heads": kv_heads,
                "norm": rng.random() < 0.5, "page": rng.choice([16, 32, 64, 128]),
                "dtype": rng.choice(["f32", "f16", "bf16"])}
    if op == "attend":
        heads, kv_heads = rng.choice([(16, 8), (32, 8), (32, 4), (64, 4), (8, 8), (12, 3), (40, 4)])
        case = {"op": op, "rows": _log_int(rng, 1, 64), "heads": heads, "kv_heads": kv_heads,
                "prefix": rng.choice([0, 1]) * _log_int(rng, 1, 8000), "own": _log_int(rng, 1, 12000),
                "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["f32", "f16", "bf16"])}
        # no drawn case reads more than the listed ones: the own parts share a budget of keys
        case["own"] = max(1, min(case["own"], 60000 // case["rows"] // max(1, kv_heads // 4)))
        return case
    return {"op": op, "rows": _log_int(rng, 1, 100), "vocab": _log_int(rng, 1000, 151936),
            "mode": rng.choice(["chat", "mixed", "open"])}


def _lengths(count, top, seed):
    """Request lengths 0 .. top, ragged, as a function of the case alone: an empty one (of several), a full one."""
    rng = random.Random(seed * 7919 + count * 31 + top)
    out = [rng.randint((top + 9) // 10, top) for _ in range(count)]
    if count > 2:
        out[count // 2] = 0
    out[0] = top
    return out


def _requests(case):
    held = _lengths(case["requests"], case["held"], 1)
    new = _lengths(case["requests"], case["new"], 2)
    return held, new


def _pages(tokens, page):
    return (tokens + page - 1) // page


# ---- inputs ------------------------------------------------------------------------------
def prepare(case, seed):
    return {"tables": _prep_tables, "append": _prep_append, "attend": _prep_attend,
            "sample": _prep_sample}[case["op"]](case, seed)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prep_tables(case, seed):
    held, new = _requests(case)
    rng = random.Random(seed)
    order = list(range(len(held)))
    rng.shuffle(order)
    held, new = [held[i] for i in order], [new[i] for i in order]
    page, n, width = case["page"], case["requests"], case["width"]
    need = sum(_pages(h + t, page) for h, t in zip(held, new))
    ids = torch.randperm(need + 37, generator=_gen(seed), device="cuda").to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    used, host = 0, np.full((n, width), -1, dtype=np.int32)
    ids_host = ids.cpu().numpy()
    for i, h in enumerate(held):  # the pages that the requests hold already
        p = _pages(h, page)
        host[i, :p] = ids_host[used:used + p]
        used += p
    table.copy_(torch.from_numpy(host))
    stride = case["new"] if case["padded"] else 0
    capacity = n * stride if stride else n * case["new"]
    state = {"case": case, "held": _ints(held), "new": _ints(new), "free": ids, "used": _ints([used]),
             "table": table, "stride": stride, "capacity": capacity, "used_out": _ints([0])}
    if own:
        from pyrite_b200.kernels import paged
        state["paged"] = paged
        state["slots"] = paged.TokenSlots.empty(n, capacity=capacity, row_stride=stride, device="cuda")
    return state


def _pool(count, kv_heads, page, dtype, gen, scale=1.0):
    return torch.randn(count, kv_heads, page, HEAD, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(
        dtype)


def _rope(max_ctx, theta=1e6):
    inv = theta ** (-2.0 * np.arange(HEAD // 2, dtype=np.float64) / HEAD)
    ang = np.arange(max_ctx, dtype=np.float64)[:, None] * inv[None, :]
    return torch.from_numpy(np.ascontiguousarray(np.stack([np.cos(ang), np.sin(ang)], axis=-1))).to("cuda")


def _prep_append(case, seed):
    g = _gen(seed)
    rows, heads, kv = case["rows"], case["heads"], case["kv_heads"]
    dtype, page = DTYPES[case["dtype"]], case["page"]
    pages = _pages(rows, page) + 3
    max_ctx = 40960
    pos = torch.randint(0, max_ctx, (rows,), generator=g, device="cuda", dtype=torch.int32)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:rows].to(torch.int32)
    if rows > 4:
        slots[rows // 3] = -1  # a finished request: nothing is stored
    state = {"case": case, "qkv": torch.randn(rows, (heads + 2 * kv) * HEAD, generator=g, device="cuda").mul_(1.5),
             "pos": pos, "slots": slots, "rope": _rope(max_ctx),
             "k": _pool(pages, kv, page, dtype, g), "v": _pool(pages, kv, page, dtype, g),
             "q_norm": torch.rand(HEAD, generator=g, device="cuda") + 0.5 if case["norm"] else None,
             "k_norm": torch.rand(HEAD, generator=g, device="cuda") + 0.5 if case["norm"] else None}
    if own:
        from pyrite_b200.kernels import paged
        state["paged"], state["pool"] = paged, paged.KVPool(state["k"], state["v"])
        state["q"] = torch.empty(rows, heads * HEAD, device="cuda")
    return state


def _prep_attend(case, seed):
    g = _gen(seed)
    rows, heads, kv, page = case["rows"], case["heads"], case["kv_heads"], case["page"]
    lens = _lengths(rows, case["own"], 3)
    random.Random(seed).shuffle(lens)
    width = _pages(case["own"], page)
    shared = _pages(case["prefix"], page)
    count = shared + sum(_pages(n, page) for n in lens) + 5
    ids = torch.randperm(count, generator=g, device="cuda").to(torch.int32)
    table = np.full((rows, width), -1, dtype=np.int32)
    ids_host, at = ids.cpu().numpy(), shared
    for i, n in enumerate(lens):
        p = _pages(n, page)
        table[i, :p] = ids_host[at:at + p]
        at += p
    dtype = DTYPES[case["dtype"]]
    k = torch.empty(count, kv, page, HEAD, dtype=dtype, device="cuda")
    v = torch.empty_like(k)
    for lo in range(0, count, 256):  # in pieces: the pools need no 32-bit copy of their size
        c = min(256, count - lo)
        k[lo:lo + c] = _pool(c, kv, page, dtype, g, 1.4)
        v[lo:lo + c] = _pool(c, kv, page, dtype, g)
    state = {"case": case, "q": torch.randn(rows, heads * HEAD, generator=g, device="cuda").mul_(1.4), "k": k, "v": v,
             "table": torch.from_numpy(table).to("cuda"), "lens": _ints(lens), "shared": ids[:shared].clone()}
    if own:
        from pyrite_b200.kernels import paged
        state["paged"], state["pool"] = paged, paged.KVPool(k, v)
        state["out"] = torch.empty(rows, heads * HEAD, device="cuda")
        state["workspace"] = paged.attention_workspace(rows, heads, kv, case["prefix"], dtype, device="cuda")
    return state


def _prep_sample(case, seed):
    g = _gen(seed)
    rows, vocab, mode = case["rows"], case["vocab"], case["mode"]
    logits = torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.2)
    # a head of likely tokens over the bulk, as a language model's logits have
    head = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
    lift = torch.rand(rows, 24, generator=g, device="cuda") * 9.0
    logits.scatter_add_(1, head, lift)
    rng = random.Random(seed)
    temp, top_k, top_p, min_p = [], [], [], []
    for j in range(rows):
        kind = {"chat": 0, "open": 4}.get(mode, j % 6)
        temp.append([0.7, 0.0, 1.0, 1.3, rng.uniform(0.7, 1.2), 0.9][kind])
        top_k.append([40, 0, 0, 1000, 0, rng.randint(2, 200)][kind])
        top_p.append([0.95, 1.0, 1.0, 0.99, rng.uniform(0.8, 0.99), 1.0][kind])
        min_p.append([0.0, 0.0, 0.0, 0.0, 0.0, 0.05][kind])
        if kind == 5:  # a constrained request: most of the vocabulary is masked
            logits[j].masked_fill_(torch.rand(vocab, generator=g, device="cuda") < 0.9, float("-inf"))
    f = lambda x: torch.tensor(x, dtype=torch.float32, device="cuda")  # noqa: E731
    state = {"case": case, "logits": logits, "u": torch.rand(rows, generator=g, device="cuda"), "temp": f(temp),
             "top_k": _ints(top_k), "top_p": f(top_p), "min_p": f(min_p)}
    if own:
        from pyrite_b200.kernels import sampling
        state["sampling"] = sampling
        state["ids"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        state["probs"] = torch.empty(rows, device="cuda")
    return state


# ---- one pass ----------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"tables": _own_tables, "append": _own_append, "attend": _own_attend, "sample": _own_sample}[op](state)
    return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[op](
        state)


def _own_tables(s):
    t = s["paged"].page_tables(s["held"], s["new"], s["case"]["page"], s["free"], s["used"], s["table"], s["slots"],
                               used_out=s["used_out"])
    out = [t.slots, t.positions, t.kv_lens, s["table"], s["used_out"]]
    return out if s["stride"] else out + [t.starts]


def _own_append(s):
    c = s["case"]
    q = s["paged"].append_kv(s["qkv"], s["pool"], s["slots"], s["pos"], s["rope"], c["heads"], q_norm=s["q_norm"],
                             k_norm=s["k_norm"], eps=EPS, q_out=s["q"])
    return [q, s["k"], s["v"]]


def _own_attend(s):
    c = s["case"]
    return s["paged"].attention(s["q"], s["pool"], s["table"], s["lens"], prefix_pages=s["shared"],
                                prefix_len=c["prefix"], out=s["out"], workspace=s["workspace"])


def _own_sample(s):
    ids, probs = s["sampling"].sample_rows(s["logits"], s["u"], s["temp"], top_k=s["top_k"], top_p=s["top_p"],
                                           min_p=s["min_p"], out=s["ids"], probs=s["probs"])
    return [ids, probs]


def _plain_tables(s):
    page, free, table = s["case"]["page"], s["free"], s["table"]
    held, new = s["held"].long(), s["new"].long()
    n, width = table.shape
    has, want = (held + page - 1) // page, (held + new + page - 1) // page
    need = want - has
    end = torch.cumsum(need, 0)
    first = end - need
    used = s["used"].long()
    col = torch.arange(width, device="cuda")
    fresh = (col >= has[:, None]) & (col < want[:, None])
    at = (used + first)[:, None] + col - has[:, None]
    table = torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table)
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), torch.cumsum(new, 0)])
    if s["stride"]:
        t = torch.arange(s["stride"], device="cuda").repeat(n)
        row = torch.arange(n, device="cuda").repeat_interleave(s["stride"])
        live = t < new[row]
    else:
        flat = torch.arange(s["capacity"], device="cuda")
        row = (torch.searchsorted(starts, flat, right=True) - 1).clamp(0, n - 1)
        t = flat - starts[row]
        live = flat < starts[-1]
    pos = held[row] + t
    slot = table[row, (pos // page).clamp(0, width - 1)].long() * page + pos % page
    none = torch.full_like(pos, -1)
    out = [torch.where(live, slot, none).int(), torch.where(live, pos, none).int(), (held + new).int(), table,
           (used + end[-1]).int()]
    return out if s["stride"] else out + [starts.int()]


def _rotate(x, cs):
    half = HEAD // 2
    a, b = x[..., :half], x[..., half:]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_append(s):
    c = s["case"]
    heads, kv, page, rows = c["heads"], c["kv_heads"], c["page"], c["rows"]
    x = s["qkv"].view(rows, heads + 2 * kv, HEAD)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    if s["q_norm"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"]
    cs = s["rope"][s["pos"].long()].float()
    q, k = _rotate(q, cs), _rotate(k, cs)
    live = (s["slots"] >= 0).nonzero()[:, 0]
    slots = s["slots"].long()[live]
    s["k"][slots // page, :, slots % page] = k[live].to(s["k"].dtype)
    s["v"][slots // page, :, slots % page] = v[live].to(s["v"].dtype)
    return [q.reshape(rows, heads * HEAD), s["k"], s["v"]]


def _plain_attend(s):
    c = s["case"]
    rows, heads, kv, page, prefix = c["rows"], c["heads"], c["kv_heads"], c["page"], c["prefix"]
    group, width = heads // kv, s["table"].shape[1]
    q = s["q"].view(rows, kv, group, HEAD) * (1.0 / math.sqrt(HEAD))

    def rows_of(pool, ids):  # the pages' tokens in order, kv heads first: (..., kv, tokens, HEAD)
        x = pool[ids.long()].float().movedim(-3, -4)
        return x.reshape(*x.shape[:-3], x.shape[-3] * x.shape[-2], HEAD)

    ids = s["table"].clamp(min=0)
    own_k, own_v = rows_of(s["k"], ids), rows_of(s["v"], ids)
    score = torch.matmul(q, own_k.transpose(-1, -2))
    live = torch.arange(width * page, device="cuda") < s["lens"][:, None]
    score = score.masked_fill(~live[:, None, None, :], float("-inf"))
    if prefix:
        pre_k, pre_v = rows_of(s["k"], s["shared"])[:, :prefix], rows_of(s["v"], s["shared"])[:, :prefix]
        flat = q.permute(1, 0, 2, 3).reshape(kv, rows * group, HEAD)
        pre = torch.matmul(flat, pre_k.transpose(-1, -2)).view(kv, rows, group, prefix).permute(1, 0, 2, 3)
        score = torch.cat([pre, score], -1)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(w[..., prefix:], own_v)
    if prefix:
        flat = w[..., :prefix].permute(1, 0, 2, 3).reshape(kv, rows * group, prefix)
        out = out + torch.matmul(flat, pre_v).view(kv, rows, group, HEAD).permute(1, 0, 2, 3)
    return out.reshape(rows, heads * HEAD)


def _plain_sample(s):
    logits = s["logits"]
    rows, vocab = logits.shape
    order, idx = torch.sort(logits, dim=-1, descending=True, stable=True)  # ties: the lowest id first
    greedy = s["temp"] <= 0
    temp = torch.where(greedy, torch.ones_like(s["temp"]), s["temp"]).double()
    w = torch.exp((order.double() - order[:, :1].double()) / temp[:, None])  # 64 bits: the border of u is sharp
    cum = torch.cumsum(w, -1)
    before = cum - w
    rank = torch.arange(vocab, device="cuda")
    k = torch.where(s["top_k"] > 0, s["top_k"].clamp(max=vocab), vocab).long()
    mass = cum.gather(1, (k - 1)[:, None])[:, 0]
    p = s["top_p"].double().clamp(0.0, 1.0)
    keep = rank < k[:, None]
    keep &= (p >= 1.0)[:, None] | (before < (p * mass)[:, None]) | (rank == 0)
    keep &= w >= s["min_p"].double().clamp(0.0, 1.0)[:, None]
    keep &= ~greedy[:, None] | (rank == 0)
    count = keep.sum(-1)
    total = cum.gather(1, (count - 1)[:, None])
    at = torch.minimum((cum <= s["u"].double()[:, None] * total).sum(-1), count - 1)[:, None]
    return [idx.gather(1, at)[:, 0].int(), (w.gather(1, at) / total)[:, 0].float()]


# ---- what a pass cannot do without ---------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "tables":
        held, new = _requests(case)
        page = case["page"]
        n, tokens = case["requests"], case["requests"] * case["new"]
        fresh = sum(_pages(h + t, page) - _pages(h, page) for h, t in zip(held, new))
        return {"bytes": n * 12 + fresh * 8 + tokens * 8, "flops": tokens * 4}
    if op == "append":
        rows, heads, kv = case["rows"], case["heads"], case["kv_heads"]
        read = rows * (heads + 2 * kv) * HEAD * 4 + rows * (HEAD // 2) * 16 + rows * 8
        write = rows * heads * HEAD * 4 + rows * 2 * kv * HEAD * ITEM[case["dtype"]]
        return {"bytes": read + write, "flops": rows * (heads + kv) * HEAD * 7}
    if op == "attend":
        rows, heads, kv, page = case["rows"], case["heads"], case["kv_heads"], case["page"]
        lens = _lengths(rows, case["own"], 3)
        keys = case["prefix"] + sum(lens)
        pages = _pages(case["prefix"], page) + sum(_pages(n, page) for n in lens)
        pairs = heads * (rows * case["prefix"] + sum(lens))
        return {"bytes": keys * kv * HEAD * 2 * ITEM[case["dtype"]] + pages * 4 + rows * heads * HEAD * 8,
                "flops": pairs * HEAD * 4}
    return {"bytes": case["rows"] * case["vocab"] * 4 + case["rows"] * 28, "flops": case["rows"] * case["vocab"] * 8}


# ---- the definitions in 64 bits --------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "append": _exact_append, "attend": _exact_attend,
            "sample": _exact_sample}[case["op"]](s)


def _exact_tables(s):
    page, stride = s["case"]["page"], s["stride"]
    held, new, free = s["held"].tolist(), s["new"].tolist(), s["free"].tolist()
    table, used = s["table"].cpu().numpy().astype(np.int64), s["used"].item()
    slots = np.full(s["capacity"], -1, dtype=np.int64)
    positions, starts = slots.copy(), [0]
    for i, (h, t) in enumerate(zip(held, new)):
        for p in range(-(-h // page), -(-(h + t) // page)):
            table[i, p] = free[used]
            used += 1
        at = i * stride if stride else starts[-1]
        for j in range(t):
            slots[at + j] = table[i, (h + j) // page] * page + (h + j) % page
            positions[at + j] = h + j
        starts.append(starts[-1] + t)
    out = [slots, positions, np.array(held) + np.array(new), table, np.array([used])]
    out = [torch.from_numpy(x).int().to("cuda") for x in (out if stride else out + [np.array(starts)])]
    return out


def _exact_append(s):
    c = s["case"]
    heads, kv, page, half = c["heads"], c["kv_heads"], c["page"], HEAD // 2
    x = s["qkv"].double().reshape(c["rows"], -1, HEAD)
    freq = torch.tensor([1e6 ** (-2.0 * i / HEAD) for i in range(half)], dtype=torch.float64, device="cuda")
    angle = s["pos"].double()[:, None] * freq
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]  # the pair (i, i + 64) as one complex number

    def head(y, weight):
        if weight is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / HEAD + EPS).sqrt() * weight.double()
        z = torch.complex(y[..., :half].contiguous(), y[..., half:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    q = head(x[:, :heads], s["q_norm"])
    k, v = head(x[:, heads:heads + kv], s["k_norm"]), x[:, heads + kv:]
    out_k, out_v = s["k"].double(), s["v"].double()
    for j, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            out_k[slot // page, :, slot % page] = k[j]
            out_v[slot // page, :, slot % page] = v[j]
    return [q.reshape(c["rows"], -1), out_k, out_v]


def _exact_attend(s):
    c = s["case"]
    heads, kv, page, prefix = c["heads"], c["kv_heads"], c["page"], c["prefix"]
    group = heads // kv
    shared = s["shared"].tolist()
    out = torch.zeros(c["rows"], heads, HEAD, dtype=torch.float64, device="cuda")
    lens, table = s["lens"].tolist(), s["table"].tolist()

    def tokens(pool, ids, n):
        return torch.cat([pool[p] for p in ids], 1)[:, :n].double() if n else None

    pk, pv = tokens(s["k"], shared, prefix), tokens(s["v"], shared, prefix)
    for b, n in enumerate(lens):
        ids = table[b][:-(-n // page)]
        k = [x for x in (pk, tokens(s["k"], ids, n)) if x is not None]
        v = [x for x in (pv, tokens(s["v"], ids, n)) if x is not None]
        if not k:
            continue
        k, v = torch.cat(k, 1), torch.cat(v, 1)
        q = s["q"][b].double().view(kv, group, HEAD)
        p = torch.softmax(torch.einsum("hgd,htd->hgt", q, k) / math.sqrt(HEAD), -1)
        out[b] = torch.einsum("hgt,htd->hgd", p, v).reshape(heads, HEAD)
    return out.reshape(c["rows"], heads * HEAD)


def _exact_sample(s):
    logits = s["logits"].double().cpu().numpy()
    temp, top_p, min_p, u = (s[k].double().cpu().numpy() for k in ("temp", "top_p", "min_p", "u"))
    top_k = s["top_k"].cpu().numpy()
    ids, probs = [], []
    for j in range(logits.shape[0]):
        row = logits[j]
        order = np.lexsort((np.arange(row.size), -row))
        if temp[j] <= 0:
            ids.append(int(order[0]))
            probs.append(1.0)
            continue
        w = np.exp((row[order] - row[order[0]]) / temp[j])
        if top_k[j] > 0:
            w = w[:top_k[j]]
        n = w.size
        if top_p[j] < 1:
            n = min(n, 1 + int(np.searchsorted(np.cumsum(w), top_p[j] * w.sum(), side="left")))
        w = w[:n]
        w = w[w >= min_p[j]]
        cum = np.cumsum(w)
        at = min(int(np.searchsorted(cum, u[j] * cum[-1], side="right")), w.size - 1)
        ids.append(int(order[at]))
        probs.append(float(w[at] / cum[-1]))
    return [torch.tensor(ids, dtype=torch.int32, device="cuda"),
            torch.tensor(probs, dtype=torch.float64, device="cuda")]
