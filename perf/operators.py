"""The operators of a speculative decoding step over a paged cache, as timed cases.

A step takes, for each sequence, the last accepted token and its drafts (a chain, or a tree in which each row names its
parent) through the model at once:

  rope     per-head norms of queries and keys, the position rotation, and the store of keys and values into the cache
  attn     attention of those rows over the cached tokens and their own ancestors
  softmax  probabilities of logits at a temperature (0: all on the largest)
  verify   which drafts the target's probabilities accept, and the token after them, from given random numbers
  fork     pages of the cache: the forks of the last step freed, sequences forked, room for the next rows (shared pages
           that would be written are copied)
  compact  the rows of the accepted drafts moved behind the tokens already cached

With `own` false every operator is computed by elementary torch operations; with `own` true by the framework's calls.
"""
import math
import random

import torch

own = False

F32, F16, BF16 = 0, 1, 30
DTYPES = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
SIZE = {F32: 4, F16: 2, BF16: 2}
# the largest listed case of each kind; a drawn one costs no more
ATTN_MOST = 16 * 98304 * 2 * 128
PREFILL_MOST = 2048 * 4096 * 16 * 128
ROWS_MOST = 8192 * 2560
SOFTMAX_MOST = 1088 * 131072
VERIFY_MOST = 64 * 17 * 131072
PAGE_MOST = 56 * 8 * 64 * 4 * 128


def _cached(name, kind, sequences, rows, context, q_heads, kv_heads, dim, typ, page, tree=False, ragged=False, layers=1):
    """A batch of `sequences` with up to `rows` rows each, over caches of up to `context` tokens."""
    return {"name": name, "kind": kind, "sequences": sequences, "rows": rows, "context": context, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "type": typ, "page": page, "tree": tree, "ragged": ragged, "layers": layers}


def _rope(case, rope, interleaved=False, gated=False):
    return case | {"rope": rope, "interleaved": interleaved, "gated": gated}


def listed():
    return [
        # one decoded token of one sequence: the smallest call, where the launch counts
        _rope(_cached("rope_1tok", "rope", 1, 1, 1000, 16, 2, 128, F16, 64), 128),
        # a prompt chunk at the largest batch, packed with an output gate, a quarter of each head rotated, far positions
        _rope(_cached("rope_prefill_8192", "rope", 1, 8192, 90000, 16, 2, 128, BF16, 64), 32, gated=True),
        # one decoded token over a short cache, wide heads
        _cached("attn_1tok", "attn", 1, 1, 500, 16, 4, 256, F16, 64),
        # one sequence's longest verify batch over a long cache, drafted as a tree, groups of five heads
        _cached("attn_tree17_24k", "attn", 1, 17, 24576, 20, 4, 128, BF16, 64, tree=True),
        # a server's batch at the largest context: the cache alone is 1.2 GB
        _cached("attn_verify17_16seq_98k", "attn", 16, 17, 98304, 16, 2, 128, F16, 64, ragged=True),
        # a 2048-token prompt chunk behind as many cached tokens
        _cached("attn_prefill_2048", "attn", 1, 2048, 2048, 16, 2, 128, BF16, 128),
        # logits of the longest verify batch
        {"name": "softmax_17x151936", "kind": "softmax", "rows": 17, "cols": 151936, "temperature": 0.7},
        # 64 sequences' verify batches
        {"name": "softmax_1088x131072", "kind": "softmax", "rows": 1088, "cols": 131072, "temperature": 1.0},
        # a chain of 16 sampled drafts of one sequence
        {"name": "verify_1seq", "kind": "verify", "sequences": 1, "rows": 17, "cols": 151936, "tree": False, "ragged": False, "greedy": False},
        # drafted trees of 64 sequences
        {"name": "verify_tree_64seq", "kind": "verify", "sequences": 64, "rows": 17, "cols": 131072, "tree": True, "ragged": True, "greedy": False},
        # eight prompts, seven further samples forked from each
        _cached("fork_8x7", "fork", 8, 17, 4000, 0, 4, 128, BF16, 64, ragged=True, layers=8) | {"fan": 7},
        # the accepted rows of sixteen trees, in every layer of a stack
        _cached("compact_16seq", "compact", 16, 17, 2000, 0, 2, 128, F16, 64, tree=True, ragged=True, layers=48),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("rope", "attn", "attn", "attn", "softmax", "verify", "fork", "compact"))
    if kind == "softmax":
        cols = _log(rng, 1000, 200000)
        return {"kind": kind, "rows": max(1, min(_log(rng, 1, 1088), SOFTMAX_MOST // cols)), "cols": cols,
                "temperature": rng.choice((0.0, 0.6, 0.7, 1.0, 1.0, 1.3))}
    if kind == "verify":
        cols, rows = _log(rng, 1000, 200000), rng.randint(2, 33)
        return {"kind": kind, "sequences": max(1, min(_log(rng, 1, 64), VERIFY_MOST // (rows * cols))), "rows": rows, "cols": cols,
                "tree": rng.random() < 0.5, "ragged": rng.random() < 0.7, "greedy": rng.random() < 0.3}
    kv_heads, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128, 256))
    q_heads, page = kv_heads * rng.choice((1, 4, 5, 8, 8, 16)), rng.choice((8, 16, 32, 64, 128, 256))
    while q_heads * dim > 5120:  # the widest row of queries
        q_heads = max(kv_heads, q_heads // 2 // kv_heads * kv_heads)
    typ, ragged = rng.choice((F16, BF16, BF16, F32)), rng.random() < 0.7
    if kind == "rope":
        rows = _log(rng, 1, 8192)
        sequences = _log(rng, 1, 64) if rows <= 64 else 1
        rows = max(1, min(rows, ROWS_MOST // (sequences * max(1, q_heads + 2 * kv_heads) * dim)))
        case = _cached("", kind, sequences, rows, _log(rng, 1, 98304 // sequences), q_heads, kv_heads, dim, typ, page,
                       tree=1 < rows <= 64 and rng.random() < 0.5, ragged=ragged, layers=rng.choice((1, 2)))
        case = _rope(case, rng.choice((dim, dim, dim // 2, dim // 4)), rng.random() < 0.5, rng.random() < 0.3)
    elif kind == "attn":
        if rng.random() < 0.2:  # a prompt chunk
            rows, context = _log(rng, 65, 2048), _log(rng, 1, 4096)
            rows = max(65, min(rows, PREFILL_MOST // ((context + rows) * q_heads * dim)))
            case = _cached("", kind, 1, rows, context, q_heads, kv_heads, dim, typ, page)
        else:
            sequences, rows = _log(rng, 1, 32), rng.choice((1, 1, 2, 5, 9, 17, 17, 33, 64))
            # room for the cache, and for what the rows have to compute
            per = sequences * kv_heads * dim * SIZE[typ] // 2
            most = min(98304, ATTN_MOST // per, 2 * PREFILL_MOST // (sequences * rows * q_heads * dim))
            case = _cached("", kind, sequences, rows, _log(rng, 1, max(2, most)), q_heads, kv_heads, dim, typ, page,
                           tree=rows > 1 and rng.random() < 0.5, ragged=ragged)
    else:
        sequences, layers = _log(rng, 1, 16), rng.choice((1, 2, 8, 16))
        fan = rng.randint(1, 7)
        if kind == "fork":
            while sequences > 1 and sequences * fan * layers * page * kv_heads * dim > PAGE_MOST:
                sequences -= 1
            while fan > 1 and sequences * fan * layers * page * kv_heads * dim > PAGE_MOST:
                fan -= 1
            layers = max(1, min(layers, PAGE_MOST // (sequences * fan * page * kv_heads * dim)))
        most = max(2, (1 << 28) // (sequences * layers * kv_heads * dim * SIZE[typ]))
        case = _cached("", kind, sequences, rng.randint(2, 33), _log(rng, 1, min(8192, most)), 0, kv_heads, dim, typ, page,
                       tree=kind == "compact", ragged=ragged, layers=layers)
        if kind == "fork":
            case |= {"fan": fan}
    return {k: v for k, v in case.items() if k != "name"}


# ---------------- inputs ----------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _counts(case, sequences):
    """How many rows and cached tokens each sequence has: `ragged` ones differ, the same way for every seed."""
    rng = random.Random(sequences * 7919 + case["rows"])
    rows, context = [case["rows"]] * sequences, [case.get("context", 0)] * sequences
    if case["ragged"]:
        rows = [case["rows"]] + [rng.randint(1, case["rows"]) for _ in range(sequences - 1)]
        context = [case.get("context", 0)] + [rng.randint(case.get("context", 0) // 2, case.get("context", 0)) for _ in range(sequences - 1)]
    return rows, context


def _parents(case, rng, rows):
    """The parent of every row: mostly the row before, else one of the few before that (a beam of drafts)."""
    out = []
    for n in rows:
        out += [-1] + [i - 1 if rng.random() < 0.5 else rng.randint(max(0, i - 5), i - 1) for i in range(1, n)]
    return out


def _batch(case, rng, rows):
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    return {"total": start[-1], "most": max(rows), "start": _ints(start), "parent": _ints(_parents(case, rng, rows)) if case["tree"] else None}


def _cache(case, gen, rows, context, spare=0, extra=0):
    """A cache whose sequences hold `context` tokens and have pages for `rows` more, in random order; `spare` pages are free,
    `extra` sequences are empty."""
    P, B = case["page"], len(context)
    need = [-(-(c + r) // P) for c, r in zip(context, rows)]
    pages, width = sum(need) + spare, max(need) + 1
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((B + extra, width), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    refs[order[:at].long()] = 1
    shape = (case["layers"], pages, case["kv_heads"], P, case["dim"])
    k, v = (torch.empty(shape, dtype=DTYPES[case["type"]], device="cuda") for _ in range(2))
    for t in (k, v):
        for i in range(case["layers"]):
            t[i].normal_(generator=gen)
    return {"k": k, "v": v, "table": table, "refs": refs, "length": _ints(list(context) + [0] * extra)}


def _logits(gen, rows, cols):
    """Logits as a language model has them: most tokens far below the best few."""
    return _normal(gen, rows, cols).mul_(4)


def prepare(case, seed):
    gen, rng = _generator(seed), random.Random(int(seed) * 7919 + 5)
    s = {"case": dict(case)}
    if case["kind"] == "softmax":
        x = _logits(gen, case["rows"], case["cols"])
        return s | {"x": x, "out": torch.empty_like(x)}
    if case["kind"] == "verify":
        B, V = case["sequences"], case["cols"]
        rows, _ = _counts(case, B)
        s |= _batch(case, rng, rows)
        N = s["total"]
        # the draft model's logits are the target's with an error
        target = _logits(gen, N, V)
        draft = torch.softmax(target + 0.7 * _normal(gen, N, V), -1)
        s["p"] = torch.softmax(target, -1)
        del target
        parent = s["parent"].tolist() if s["parent"] is not None else None
        up, rank, first = [], [], 0
        for n in rows:  # the row whose distribution each draft was drawn from, and its place among its siblings
            seen = [0] * n
            for i in range(n):
                j = 0 if i == 0 else (parent[first + i] if parent else i - 1)
                up.append(first + j)
                rank.append(seen[j] if i else 0)
                seen[j] += 1 if i else 0
            first += n
        up, rank = torch.tensor(up, device="cuda"), torch.tensor(rank, device="cuda")
        if case["greedy"]:  # a row's drafts are the draft model's best tokens, one each
            best = torch.topk(draft, min(V, 34), -1).indices
            s["token"] = best[up, rank].int()
            s["q"] = None
        else:
            s["token"] = torch.cat([torch.multinomial(draft[up[i:i + 64]], 1, generator=gen)[:, 0] for i in range(0, N, 64)]).int()
            s["q"] = draft
        s["u"] = torch.rand(N, generator=gen, device="cuda")
        s["u_last"] = torch.rand(B, generator=gen, device="cuda")
        s["tokens_out"], s["path"] = (torch.full((B, s["most"]), -1, dtype=torch.int32, device="cuda") for _ in range(2))
        s["count"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        return s
    rows, context = _counts(case, case["sequences"])
    if case["kind"] == "fork":
        fan, B = case["fan"], case["sequences"]
        s |= _cache(case, gen, [0] * B, context, spare=B * (fan + 1) * (-(-case["rows"] // case["page"]) + 2), extra=B * fan)
        s["table"] = torch.nn.functional.pad(s["table"], (0, -(-case["rows"] // case["page"]) + 1), value=-1).contiguous()
        s["src"] = _ints([b for b in range(B) for _ in range(fan)])
        s["dst"] = _ints(list(range(B, B * (fan + 1))))
        # what is kept of each sequence: all of the prompts, nothing of the forks
        s["keep"] = _ints(list(context) + [0] * (B * fan))
        more, _ = _counts(case, B * (fan + 1))
        s |= _batch(case, rng, more)
        s["status"] = torch.zeros(B * (fan + 1), dtype=torch.int32, device="cuda")
        return s
    s |= _batch(case, rng, rows) | _cache(case, gen, rows, context, spare=3)
    N, Hq, Hkv, D = s["total"], case["q_heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "compact":
        # a branch is accepted whose rows lie behind those of the branches that were tried before it
        path, count = [], []
        for n in rows:
            m = rng.randint(1, max(1, n // 3))
            same = rng.randint(1, m)
            behind = sorted(rng.sample(range(m, n), min(m - same, n - m)))
            kept = list(range(same)) + behind
            kept = kept if len(kept) == m else list(range(m))
            path.append(kept + [-1] * (s["most"] - m))
            count.append(m)
        return s | {"path": _ints(path), "count": _ints(count), "new_length": torch.zeros_like(s["length"])}
    if case["kind"] == "attn":
        return s | {"q": _normal(gen, N, Hq, D), "out": torch.empty(N, Hq, D, device="cuda")}
    # rope: one packed projection per row, q heads (each followed by its output gate where gated), then k and v heads
    Wq = D * (2 if case["gated"] else 1)
    qkv = _normal(gen, N, Hq * Wq + 2 * Hkv * D)
    i = torch.arange(case["rope"] // 2, dtype=torch.float64, device="cuda")
    return s | {"qkv": qkv, "q_norm": 1 + 0.1 * _normal(gen, D), "k_norm": 1 + 0.1 * _normal(gen, D),
                "freq": torch.exp(-math.log(1e6) * 2 * i / case["rope"]), "out": torch.empty(N, Hq, D, device="cuda")}


# ---------------- the framework's calls ----------------

def _plan(s):
    """Descriptors and workspace, which a program keeps with its buffers."""
    if "plan" in s:
        return s["plan"]
    import ctypes
    from nebula_amd import qg
    c, plan = s["case"], {}

    def ptr(name):
        return s[name].data_ptr() if s.get(name) is not None else None
    if "start" in s:
        plan["batch_"] = qg.KvBatch(rows=s["total"], max_rows=s["most"], start=ptr("start"), parent=ptr("parent"))
        plan["batch"] = ctypes.byref(plan["batch_"])
    if "k" in s:
        plan["cache_"] = qg.KvCache(k=ptr("k"), v=ptr("v"), type=c["type"], layers=c["layers"], pages=s["k"].shape[1], kv_heads=c["kv_heads"],
                                    page_tokens=c["page"], head_dim=c["dim"], refs=ptr("refs"), table=ptr("table"), length=ptr("length"),
                                    sequences=s["length"].numel(), table_pages=s["table"].shape[1])
        plan["cache"] = ctypes.byref(plan["cache_"])
    lib = qg.lib()
    plan["bytes"] = {"softmax": lambda: lib.qg_softmax_workspace_bytes(c["rows"], c["cols"]),
                     "verify": lambda: lib.qg_verify_workspace_bytes(c["sequences"], c["cols"]),
                     "attn": lambda: lib.qg_tree_attention_workspace_bytes(plan["cache"], plan["batch"], c["q_heads"]),
                     "fork": lambda: lib.qg_kv_workspace_bytes(plan["cache"]),
                     "compact": lambda: 0, "rope": lambda: 0}[c["kind"]]()
    plan["ws_"] = torch.empty(max(16, plan["bytes"]), dtype=torch.uint8, device="cuda")
    plan["ws"] = plan["ws_"].data_ptr()
    if c["kind"] == "rope":
        D, Hq, Hkv, x = c["dim"], c["q_heads"], c["kv_heads"], s["qkv"]
        Wq, row = D * (2 if c["gated"] else 1), x.shape[1]
        at = x.data_ptr()
        plan["rows_"] = qg.QkRows(q=at, k=at + 4 * Hq * Wq, v=at + 4 * (Hq * Wq + Hkv * D), q_row=row, q_head=Wq, k_row=row, k_head=D,
                                  v_row=row, v_head=D, rows=s["total"], q_heads=Hq, kv_heads=Hkv, head_dim=D, q_norm=ptr("q_norm"),
                                  k_norm=ptr("k_norm"), eps=1e-6, rope_dims=c["rope"], interleaved=int(c["interleaved"]), freq=ptr("freq"),
                                  position=None)
        plan["rows"] = ctypes.byref(plan["rows_"])
    s["plan"] = plan
    return plan


def _own(s):
    from nebula_amd import qg
    c, p = s["case"], _plan(s)

    def at(name):
        return s[name].data_ptr() if s[name] is not None else None
    if c["kind"] == "softmax":
        qg.call("softmax", at("out"), at("x"), c["rows"], c["cols"], c["temperature"], p["ws"], p["bytes"])
    elif c["kind"] == "verify":
        qg.call("verify_drafts", at("tokens_out"), at("path"), at("count"), at("p"), at("q"), at("token"), at("u"), at("u_last"),
                c["cols"], c["sequences"], p["batch"], p["ws"], p["bytes"])
    elif c["kind"] == "attn":
        qg.call("tree_attention", at("out"), at("q"), c["q_heads"], c["dim"] ** -0.5, p["cache"], 0, p["batch"], p["ws"], p["bytes"])
    elif c["kind"] == "rope":
        qg.call("qk_norm_rope", at("out"), None, p["rows"], p["cache"], c["layers"] - 1, p["batch"])
    elif c["kind"] == "compact":
        qg.call("kv_compact", p["cache"], p["batch"], at("path"), at("count"), at("new_length"))
    else:
        qg.call("kv_truncate", p["cache"], at("keep"))
        qg.call("kv_fork", p["cache"], at("dst"), at("src"), s["dst"].numel(), p["ws"], p["bytes"])
        qg.call("kv_reserve", p["cache"], p["batch"], at("status"), p["ws"], p["bytes"])


# ---------------- the plain forms ----------------

def _row_places(s):
    """The sequence of every row and the row's place in it."""
    i = torch.arange(s["total"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["start"], i, right=True) - 1
    return seq, (i - s["start"][seq]).long()


def _ancestors(s, seq, place):
    """[rows, most] whether a row of the same sequence is on the row's way to the root, itself included."""
    seen = torch.zeros(s["total"], s["most"] + 1, dtype=torch.bool, device="cuda")
    if s["parent"] is None:
        seen[:, :-1] = torch.arange(s["most"], device="cuda") <= place[:, None]
        return seen[:, :-1]
    first, parent, at = s["start"][seq].long(), s["parent"].long(), place
    for _ in range(s["most"]):
        seen.scatter_(1, torch.where(at >= 0, at, s["most"])[:, None], True)
        at = torch.where(at >= 0, parent[first + at.clamp_min(0)], at)
    return seen[:, :-1]


def _rows_into(s, seq, slot, k, v):
    """Stores rows k, v [rows, heads, dim] at token `slot` of their sequences, in the case's layer."""
    P, layer = s["case"]["page"], s["case"]["layers"] - 1
    page = s["table"][seq, slot // P].long()
    s["k"][layer, page, :, slot % P] = k.to(s["k"].dtype)
    s["v"][layer, page, :, slot % P] = v.to(s["v"].dtype)


def _plain_rope(s):
    c = s["case"]
    D, Hq, Hkv, R, N = c["dim"], c["q_heads"], c["kv_heads"], c["rope"], s["total"]
    Wq = D * (2 if c["gated"] else 1)
    q = s["qkv"][:, :Hq * Wq].reshape(N, Hq, Wq)[:, :, :D]
    k, v = s["qkv"][:, Hq * Wq:].reshape(N, 2, Hkv, D).unbind(1)
    seq, place = _row_places(s)
    depth = place if s["parent"] is None else _ancestors(s, seq, place).sum(-1) - 1
    length = s["length"][seq]
    angle = (length + depth).double()[:, None] * s["freq"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        a, b = (x[..., 0:R:2], x[..., 1:R:2]) if c["interleaved"] else (x[..., :R // 2], x[..., R // 2:R])
        y, z = a * cos - b * sin, b * cos + a * sin
        y = torch.stack((y, z), -1).flatten(-2) if c["interleaved"] else torch.cat((y, z), -1)
        return torch.cat((y, x[..., R:]), -1)
    s["out"].copy_(turned(q, s["q_norm"]))
    _rows_into(s, seq, length + place, turned(k, s["k_norm"]), v)


def _plain_attn(s):
    c = s["case"]
    B, n, Hq, Hkv, D, P = c["sequences"], s["most"], c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    L, G = s["table"].shape[1] * P, Hq // Hkv

    def gathered(pool):
        return pool[0][s["table"].clamp_min(0).long()].transpose(1, 2).reshape(B, Hkv, L, D).float()
    first, count = s["start"][:-1].long(), (s["start"][1:] - s["start"][:-1]).long()
    i = torch.arange(n, device="cuda")
    row = (first[:, None] + i).clamp_max(s["total"] - 1)
    q = s["q"][row].reshape(B, n, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * G, D)
    scores = (q @ gathered(s["k"]).transpose(-1, -2)).mul_(D ** -0.5)
    j = torch.arange(L, device="cuda")
    length = s["length"].long()
    seq, place = _row_places(s)
    behind = j - length[:, None]  # the row of the batch that lies at each place
    seen = behind[:, None] < 0
    if s["parent"] is None:
        seen = seen | (behind[:, None] <= i[:, None])
    else:
        up = _ancestors(s, seq, place)[row]  # [B, n, most]
        up = up.gather(2, behind[:, None].clamp(0, n - 1).expand(B, n, L))
        seen = seen | (up & (behind[:, None] >= 0) & (behind[:, None] < count[:, None, None]))
    scores.view(B, Hkv, n, G, L).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    w = scores.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    out = (w @ gathered(s["v"])) / w.sum(-1, keepdim=True)
    s["out"].copy_(out.reshape(B, Hkv, n, G, D).transpose(1, 2)[seq, place].reshape(-1, Hq, D))


def _plain_softmax(s):
    T, x = s["case"]["temperature"], s["x"]
    if T == 0:
        s["out"].zero_().scatter_(1, x.argmax(-1, keepdim=True), 1.0)
        return
    e = ((x - x.amax(-1, keepdim=True)) / T).exp_()
    torch.div(e, e.sum(-1, keepdim=True), out=s["out"])


def _plain_verify(s):
    B, V, n = s["case"]["sequences"], s["case"]["cols"], s["most"]
    first, rows = s["start"][:-1].long(), s["start"][1:] - s["start"][:-1]
    b = torch.arange(B, device="cuda")
    at = torch.zeros(B, dtype=torch.long, device="cuda")  # the node that the walk has come to
    a, mass = torch.zeros(B, dtype=torch.float64, device="cuda"), torch.ones(B, dtype=torch.float64, device="cuda")
    gone = torch.zeros(B, n, dtype=torch.bool, device="cuda")  # children of the node that were rejected
    kept = torch.zeros(B, dtype=torch.int32, device="cuda")
    path, tokens = torch.full((B, n + 1), -1, dtype=torch.int32, device="cuda"), torch.full((B, n + 1), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    place = torch.arange(n, device="cuda")
    token = s["token"][(first[:, None] + place).clamp_max(s["total"] - 1)].long()

    def left():
        """The node's distribution without what its rejected children took, times a constant."""
        p = s["p"][first + at].double()
        if s["q"] is not None:
            return (p - a[:, None] * s["q"][first + at].double()).clamp_min_(0)
        drop = torch.zeros(B, V + 1, dtype=torch.bool, device="cuda").scatter_(1, torch.where(gone, token, V), True)
        return p.masked_fill_(drop[:, :-1], 0)
    for i in range(1, n):
        row = (first + i).clamp_max(s["total"] - 1)
        child = (i < rows) & ((s["parent"][row] if s["parent"] is not None else i - 1) == at)
        x = s["token"][row].long()
        p, u = s["p"][first + at, x].double(), s["u"][row].double()
        if s["q"] is not None:
            q = s["q"][first + at, x].double()
            p = (p - a * q).clamp_min(0)
            accept = child & (u * q * mass < p)
        else:
            p = p.masked_fill((gone & (token == x[:, None])).any(-1), 0)
            accept = child & (u * mass < p)
        reject = child & ~accept
        if s["q"] is not None:
            a = torch.where(reject, a + mass, a)
            mass = torch.where(reject, left().sum(-1), mass)
        else:
            mass = torch.where(reject, mass - p, mass)
            gone[:, i] |= reject
        gone &= ~accept[:, None]
        a, mass = a.masked_fill(accept, 0), mass.masked_fill(accept, 1)
        at = torch.where(accept, i, at)
        slot = torch.where(accept, kept, n).long()[:, None]
        tokens.scatter_(1, slot, x.int()[:, None])
        kept = kept + accept.int()
        path.scatter_(1, torch.where(accept, kept, n).long()[:, None], i)
    w = left()
    sums = w.cumsum(-1)
    none = ~(sums[:, -1] > 0)
    w = torch.where(none[:, None], s["p"][first + at].double(), w)
    sums = torch.where(none[:, None], w.cumsum(-1), sums)
    goal = s["u_last"].double() * sums[:, -1]
    last = V - 1 - (w > 0).flip(-1).int().argmax(-1)
    pick = torch.minimum((sums <= goal[:, None]).sum(-1), last)
    tokens[b, kept.long()] = pick.int()
    s["tokens_out"].copy_(tokens[:, :n])
    s["path"].copy_(path[:, :n])
    s["count"].copy_(kept + 1)


def _plain_compact(s):
    c, n = s["case"], s["most"]
    P, rows = c["page"], (s["start"][1:] - s["start"][:-1]).long()
    i = torch.arange(n, device="cuda")
    to = torch.minimum(i, rows[:, None] - 1)
    src = torch.where(i < s["count"][:, None], s["path"].long(), to) + s["length"][:, None]
    dst = torch.where(i < s["count"][:, None], i, to) + s["length"][:, None]
    b = torch.arange(rows.numel(), device="cuda")[:, None].expand_as(src).reshape(-1)
    src, dst = src.reshape(-1), dst.reshape(-1)
    sp, dp = s["table"][b, src // P].long(), s["table"][b, dst // P].long()
    for pool in (s["k"], s["v"]):
        pool[:, dp, :, dst % P] = pool[:, sp, :, src % P]
    s["new_length"].copy_(s["length"] + s["count"])


def _plain_fork(s):
    table, refs, length, P = s["table"], s["refs"], s["length"], s["case"]["page"]
    B, W = table.shape
    j = torch.arange(W, device="cuda")

    def count(pages, held, by):
        refs.index_add_(0, pages.clamp_min(0).reshape(-1).long(), (held.reshape(-1) * by).int())
    # free what lies behind the kept tokens
    length.copy_(torch.minimum(length, s["keep"]))
    gone = (table >= 0) & (j >= ((length + P - 1) // P)[:, None])
    count(table, gone, -1)
    table.masked_fill_(gone, -1)
    # forks share their source's pages
    src, dst = s["src"].long(), s["dst"].long()
    rows = table[src].masked_fill(j >= ((length[src] + P - 1) // P)[:, None], -1)
    count(rows, rows >= 0, 1)
    table[dst], length[dst] = rows, length[src]
    # room for the next rows: a shared page that would be written is copied, except for its first writer where no other
    # sequence holds it
    add = s["start"][1:] - s["start"][:-1]
    here, end = (length // P).long(), ((length + add + P - 1) // P).long()
    page = table.gather(1, here[:, None].clamp_max(W - 1))[:, 0].masked_fill((add <= 0) | (length % P == 0), -1)
    same = (page[:, None] == page) & (page >= 0)
    before = torch.tril(same, -1).any(-1)
    held = refs[page.clamp_min(0).long()]
    copied = (page >= 0) & (held > 1) & (before | (same.sum(-1) < held))
    fresh = (j >= here[:, None]) & (j < end[:, None]) & ((table < 0) | (copied[:, None] & (j == here[:, None])))
    free = torch.argsort((refs != 0).int(), stable=True)  # the free pages first, in order
    place = (fresh.reshape(-1).int().cumsum(0) - 1).clamp(0, free.numel() - 1)
    got = free[place].reshape(B, W).int()
    new = torch.where(fresh, got, table)
    to = new.gather(1, here[:, None].clamp_max(W - 1))[:, 0].long()
    # a sequence without a copy copies a page of its own onto itself
    own_page = table[:, 0].long().clamp_min(0)
    a, b = torch.where(copied, page.long(), own_page), torch.where(copied, to, own_page)
    for pool in (s["k"], s["v"]):
        for layer in pool:
            layer[b] = layer[a]
    count(page, copied, -1)
    count(got, fresh, 1)
    table.copy_(new)
    s["status"].zero_()


def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        _own(s)
    else:
        {"rope": _plain_rope, "attn": _plain_attn, "softmax": _plain_softmax, "verify": _plain_verify, "compact": _plain_compact,
         "fork": _plain_fork}[kind](s)
    if kind in ("softmax", "attn"):
        return s["out"]
    if kind == "rope":
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    if kind == "verify":
        return {"tokens": s["tokens_out"], "path": s["path"], "count": s["count"]}
    if kind == "compact":
        return {"k": s["k"], "v": s["v"], "length": s["new_length"]}
    return {"k": s["k"], "v": s["v"], "table": s["table"], "refs": s["refs"], "length": s["length"], "status": s["status"]}


# ---------------- what a pass needs, and its exact result ----------------

def work(case):
    kind = case["kind"]
    if kind == "softmax":
        n = case["rows"] * case["cols"]
        return {"bytes": 8 * n, "flops": 4 * n}
    part = 0.75 if case["ragged"] else 1.0  # the mean of a ragged batch's rows and lengths
    B = case["sequences"]
    if kind == "verify":  # the probabilities that the last token is drawn from
        n = B * case["cols"] * (1 if case["greedy"] else 2)
        return {"bytes": 4 * n, "flops": 3 * n}
    es, D, Hq, Hkv = SIZE[case["type"]], case["dim"], case["q_heads"], case["kv_heads"]
    mean = (case["rows"] + 1) / 2 if case["ragged"] else case["rows"]
    rows = case["rows"] + (B - 1) * mean
    if kind == "rope":
        return {"bytes": rows * D * (4 * (2 * Hq + 2 * Hkv) + 2 * es * Hkv), "flops": rows * D * 10 * (Hq + Hkv)}
    if kind == "attn":
        keys = case["context"] * (1 + (B - 1) * part) if case["ragged"] else case["context"] * B
        pairs = rows * (keys / B + (case["rows"] + 1) / 2)
        return {"bytes": (keys + rows) * Hkv * D * 2 * es + rows * Hq * D * 8, "flops": 4 * pairs * Hq * D}
    if kind == "compact":  # about half of the kept rows move
        moved = B * max(1, case["rows"] // 6) / 2
        return {"bytes": moved * case["layers"] * Hkv * D * 4 * es, "flops": 0}
    # every fork and its source write into a page that they share: one copy for each fork
    copies = 0 if case["context"] % case["page"] == 0 and not case["ragged"] else B * case["fan"]
    return {"bytes": copies * case["layers"] * case["page"] * Hkv * D * 4 * es + 8 * B * (1 + case["fan"]) * (case["context"] // case["page"] + 1), "flops": 0}


def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "compact"):
        return None  # copies and whole numbers
    s = prepare(case, seed)
    if kind == "softmax":
        if case["temperature"] == 0:
            return None
        out = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda")
        for i in range(0, case["rows"], 64):
            z = s["x"][i:i + 64].double() / case["temperature"]
            out[i:i + 64] = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
        return out
    start = s["start"].tolist()
    parent = s["parent"].tolist() if s["parent"] is not None else None
    if kind == "verify":
        return _exact_verify(s, start, parent)
    lines = []  # for each row the rows of its sequence on its way to the root
    for first, end in zip(start, start[1:]):
        for i in range(end - first):
            up = (parent[first + i] if parent else i - 1)
            lines.append((lines[first + up] if up >= 0 else []) + [i] if parent or end - first <= 64 else i)
    D, P = case["dim"], case["page"]
    if kind == "rope":
        Hq, Hkv, R = case["q_heads"], case["kv_heads"], case["rope"]
        Wq, length = D * (2 if case["gated"] else 1), s["length"].tolist()
        pos = [length[b] + (len(lines[r]) - 1 if isinstance(lines[r], list) else lines[r])
               for b in range(len(length)) for r in range(start[b], start[b + 1])]
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           torch.tensor(pos, dtype=torch.float64, device="cuda")[:, None] * s["freq"])[:, None]
        x = s["qkv"].double()

        def turned(x, w):
            x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + 1e-6) * w.double()
            head = x[..., :R]
            if case["interleaved"]:
                z = turn * torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous())
                head = torch.view_as_real(z).flatten(-2)
            else:
                z = turn * torch.complex(head[..., :R // 2], head[..., R // 2:])
                head = torch.cat((z.real, z.imag), -1)
            return torch.cat((head, x[..., R:]), -1)
        q = turned(x[:, :Hq * Wq].reshape(-1, Hq, Wq)[..., :D], s["q_norm"])
        k, v = x[:, Hq * Wq:].reshape(-1, 2, Hkv, D).unbind(1)
        k = turned(k, s["k_norm"])
        K, V, layer = s["k"].double(), s["v"].double(), case["layers"] - 1
        at = [(b, length[b] + i) for b in range(len(length)) for i in range(start[b + 1] - start[b])]
        where = torch.tensor(at, device="cuda")
        page = s["table"][where[:, 0], where[:, 1] // P].long()
        K[layer, page, :, where[:, 1] % P] = k
        V[layer, page, :, where[:, 1] % P] = v
        return {"q": q, "k": K, "v": V}
    if start[-1] * case["q_heads"] * (case["context"] + case["rows"]) * D > 4e12:
        return None
    Hq, Hkv = case["q_heads"], case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["length"].tolist()):
        first, n = start[b], start[b + 1] - start[b]
        pages = s["table"][b, :-(-(length + n) // P)].long()
        seen = torch.ones(n, length + n, dtype=torch.bool, device="cuda")
        if isinstance(lines[first], list):
            tail = torch.zeros(n, n, dtype=torch.bool)
            for i in range(n):
                tail[i, lines[first + i]] = True
            seen[:, length:] = tail.cuda()
        else:
            seen[:, length:] = torch.tril(seen[:, length:])
        for h in range(Hkv):
            K, V = (pool[0, pages, h].reshape(-1, D)[:length + n].double() for pool in (s["k"], s["v"]))
            for g in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                z = (s["q"][first:first + n, g].double() @ K.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
                out[first:first + n, g] = torch.softmax(z, -1) @ V
    return out


def _exact_verify(s, start, parent):
    B, n, V = s["case"]["sequences"], s["most"], s["case"]["cols"]
    token, u, u_last = s["token"].tolist(), s["u"].tolist(), s["u_last"].tolist()
    tokens, path, count = torch.full((B, n), -1, dtype=torch.int32), torch.full((B, n), -1, dtype=torch.int32), []
    for b in range(B):
        first, rows = start[b], start[b + 1] - start[b]
        node, way, said = 0, [0], []
        while True:
            p = s["p"][first + node].double()
            mass, total = p, 1.0  # what is left of the node's distribution
            found = None
            for i in range(1, rows):
                if (parent[first + i] if parent else i - 1) != node:
                    continue
                x = token[first + i]
                if s["q"] is not None:
                    q = s["q"][first + node].double()
                    if u[first + i] * float(q[x]) < float(mass[x]) / total:
                        found = i
                        break
                    mass, total = (mass / total - q).clamp_min(0), None
                    total = float(mass.sum())
                else:
                    if u[first + i] * total < float(mass[x]):
                        found = i
                        break
                    total -= float(mass[x])
                    mass = mass.clone()
                    mass[x] = 0
            if found is None:
                break
            way.append(found)
            said.append(token[first + found])
            node = found
        c = mass.cumsum(0)
        if not float(c[-1]) > 0:
            mass, c = p, p.cumsum(0)
        pick = int((c <= u_last[b] * float(c[-1])).sum())
        said.append(min(pick, int(torch.nonzero(mass > 0)[-1])))
        tokens[b, :len(said)], path[b, :len(way)] = _cpu(said), _cpu(way)
        count.append(len(way))
    return {"tokens": tokens.cuda(), "path": path.cuda(), "count": _ints(count)}


def _cpu(values):
    return torch.tensor(values, dtype=torch.int32)
