"""The operators of answering one prompt several times, and of drawing its tokens, as timed cases.

A server forks a prompt's pages for several samples, agents or drafts and then takes all of them on together:

  prefixes  which sequences of a batch begin with the same pages, from the tables on the device
  shared    attention of the batch's rows where pages that several sequences hold are read once for all of them
            (with the call before it that finds them, once for all layers)
  sample    tokens drawn from logits after temperature, top-k, top-p and min-p of each row, by given random numbers, with
            their log-probabilities
  probs     the probabilities that such a draw has (what drafts are drawn from and verified against)

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
SHARED_MOST = 64 * 98304 * 16 * 128
CACHE_MOST = 1 << 30
LOGITS_MOST = 1088 * 131072
PAIRS_MOST = 1024 * 1024 * 80

# temperature, top-k (0: all), top-p, min-p of a row's request
REQUESTS = [(0.7, 20, 0.8, 0.0), (1.0, 0, 1.0, 0.0), (0.6, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 50, 1.0, 0.0), (1.3, 0, 1.0, 0.05),
            (0.8, 40, 0.95, 0.05), (1.0, 0, 0.9, 0.0), (0.9, 200, 0.99, 0.0), (1.0, 1000, 0.95, 0.02)]


def _forks(name, kind, system, prompts, samples, context, tail, page, q_heads=0, kv_heads=1, dim=64, typ=F16, rows=1, tree=False,
           ragged=False, layers=1, branch=False):
    """`prompts` prompts of up to `context` tokens behind the same `system` tokens, `samples` sequences of each with up to `tail`
    tokens of their own and up to `rows` rows in the batch; `branch`: each left its prompt's text at a place of its own."""
    return {"name": name, "kind": kind, "system": system, "prompts": prompts, "samples": samples, "context": context, "tail": tail,
            "page": page, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "type": typ, "rows": rows, "tree": tree,
            "ragged": ragged, "layers": layers, "branch": branch}


def _logits(name, kind, rows, cols, requests, draws=1, masked=False, rounded=False):
    """`requests`: the places in REQUESTS that the rows go through; `masked`: a grammar allows some tokens only; `rounded`: the
    logits are those of a model in bfloat16, in which many are equal."""
    case = {"name": name, "kind": kind, "rows": rows, "cols": cols, "requests": requests, "masked": masked, "rounded": rounded}
    return case | {"draws": draws} if kind == "sample" else case


ALL = "0123456789"


def listed():
    return [
        # eight branches of one text: the smallest call, where the launches count
        _forks("prefixes_8seq", "prefixes", 0, 1, 8, 4000, 100, 64, branch=True),
        # the most sequences a cache has: 32 prompts behind one system text, 32 branches of each
        _forks("prefixes_1024seq", "prefixes", 1024, 32, 32, 4000, 100, 64, ragged=True, branch=True),
        # eight samples of a short prompt, one token each, wide heads, in every layer of a small stack
        _forks("shared_8x1_2k", "shared", 0, 1, 8, 2000, 100, 64, 16, 4, 256, F16, layers=8),
        # 64 samples of the longest prompt
        _forks("shared_64x1_98k", "shared", 0, 1, 64, 98304, 500, 64, 16, 2, 128, F16, ragged=True),
        # a drafted tree in each of sixteen samples of a long prompt, groups of five heads
        _forks("shared_tree17_16seq_24k", "shared", 0, 1, 16, 24576, 300, 64, 20, 4, 128, BF16, 17, tree=True, ragged=True),
        # a server's batch: a system text, eight prompts behind it, eight samples of each
        _forks("shared_2level_8x8", "shared", 8192, 8, 8, 8192, 1000, 128, 16, 2, 128, BF16, ragged=True),
        # one token of one sequence: the smallest call
        _logits("sample_1row", "sample", 1, 151936, "0"),
        # eight first tokens of a prompt that is answered eight times, from the same row
        _logits("sample_1row_8draws", "sample", 1, 131072, "2", draws=8, rounded=True),
        # a full server's batch, each row with its own settings
        _logits("sample_1088x131072", "sample", 1088, 131072, ALL),
        # the longest verify batch of one sequence
        _logits("probs_17x151936", "probs", 17, 151936, "0"),
        # a few sequences' drafts under a grammar, settings of their own
        _logits("probs_68x50000", "probs", 68, 50000, ALL, masked=True),
        # 64 sequences' verify batches
        _logits("probs_1088x131072", "probs", 1088, 131072, ALL),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("prefixes", "shared", "shared", "shared", "sample", "sample", "probs", "probs"))
    if kind in ("sample", "probs"):
        cols = _log(rng, 1000, 200000)
        rows = max(1, min(_log(rng, 1, 1088), LOGITS_MOST // cols))
        requests = rng.choice((ALL, ALL, rng.choice(ALL), rng.choice(ALL), "".join(rng.sample(ALL, 3))))
        case = _logits("", kind, rows, cols, requests, rng.choice((1, 1, 2, 5, 16)), rng.random() < 0.3, rng.random() < 0.4)
        return {k: v for k, v in case.items() if k != "name"}
    page, ragged = rng.choice((8, 16, 32, 64, 128, 256)), rng.random() < 0.7
    if kind == "prefixes":
        prompts = _log(rng, 1, 64)
        samples = _log(rng, 1, 1024 // prompts)
        width = max(2, min(1600, PAIRS_MOST // (prompts * samples) ** 2))
        system = rng.choice((0, _log(rng, 1, max(2, width * page // 2))))
        context = _log(rng, 1, max(2, width * page // 2))
        case = _forks("", kind, system, prompts, samples, context, _log(rng, 1, 200), page, rows=rng.choice((1, 1, 5, 17)), ragged=ragged,
                      branch=True)
        return {k: v for k, v in case.items() if k != "name"}
    kv_heads, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128, 256))
    q_heads, typ = kv_heads * rng.choice((1, 4, 5, 8, 8, 16)), rng.choice((F16, F16, BF16, BF16, F32))
    while q_heads * dim > 5120:  # the widest row of queries
        q_heads = max(kv_heads, q_heads // 2 // kv_heads * kv_heads)
    rows = rng.choice((1, 1, 1, 2, 5, 9, 17, 17, 33))
    prompts = rng.choice((1, 1, 1, 2, 4, 8))
    samples = _log(rng, 1, 64 // prompts)
    layers, tail = rng.choice((1, 1, 1, 2, 4)), _log(rng, 1, 1000)
    most = min(98304, SHARED_MOST // (prompts * samples * rows * q_heads * dim * layers),
               CACHE_MOST // (prompts * kv_heads * dim * SIZE[typ] * layers * 2))
    tail = min(tail, max(1, CACHE_MOST // (prompts * samples * kv_heads * dim * SIZE[typ] * layers * 4)), max(1, most // 4))
    context = _log(rng, 1, max(2, most // 2))
    system = rng.choice((0, _log(rng, 1, max(2, most // 4))))
    case = _forks("", kind, system, prompts, samples, context, tail, page, q_heads, kv_heads, dim, typ, rows,
                  tree=rows > 1 and rng.random() < 0.5, ragged=ragged, layers=layers, branch=rng.random() < 0.25)
    return {k: v for k, v in case.items() if k != "name"}


# ---------------- inputs ----------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 31)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _layout(case, seed=0):
    """The sequences: prompt, tokens up to its end, tokens of these that are held with it, tokens of their own behind them and rows, in
    an order as they came and went.  Where attention is computed all seeds have the same."""
    rng = random.Random(case["prompts"] * 7919 + case["samples"] * 104729 + case["context"] + (seed * 1299709 if case["kind"] == "prefixes" else 0))
    out = []
    for p in range(case["prompts"]):
        context = rng.randint((case["context"] + 1) // 2, case["context"]) if case["ragged"] and p else case["context"]
        for _ in range(case["samples"]):
            tail = rng.randint(0, case["tail"]) if case["ragged"] else case["tail"]
            rows = rng.randint(1, case["rows"]) if case["ragged"] and out else case["rows"]
            whole = case["system"] + context
            out.append((p, whole, rng.randint(whole // 4, whole) if case["branch"] else whole, tail, rows))
    rng.shuffle(out)
    return out


def _tables(case, layout, rng):
    """Page tables as forks leave them: whole pages of the system text and of a prompt are held by all that begin with them."""
    P, next_page, tables, heads = case["page"], 0, [], {}
    order = []

    def take(n):
        nonlocal next_page
        next_page += n
        return list(range(next_page - n, next_page))
    system = take(case["system"] // P)
    for p, whole, held, tail, rows in layout:
        if p not in heads:
            heads[p] = system + take(whole // P - len(system))
        same = heads[p][:held // P]
        tables.append(same + take(-(-(held + tail + rows) // P) - len(same)))
    order = list(range(next_page))
    rng.shuffle(order)  # pages lie where they were free
    width = max(len(t) for t in tables) + 1
    return [[order[x] for x in t] + [-1] * (width - len(t)) for t in tables], next_page + 2


def prepare(case, seed):
    gen, rng = _generator(seed), random.Random(int(seed) * 7919 + 11)
    s = {"case": dict(case)}
    if case["kind"] in ("sample", "probs"):
        R, V = case["rows"], case["cols"]
        x = torch.randn(R, V, generator=gen, device="cuda").mul_(4)
        if case["masked"]:
            x[:, torch.rand(V, generator=gen, device="cuda") < 0.4] = -math.inf
        if case["rounded"]:
            x = x.bfloat16().float()
        ask = [REQUESTS[int(case["requests"][i % len(case["requests"])])] for i in range(R)]
        for i, (what, off, typ) in enumerate((("temperature", 1.0, torch.float32), ("top_k", 0, torch.int32), ("top_p", 1.0, torch.float32),
                                              ("min_p", 0.0, torch.float32))):
            values = [a[i] for a in ask]
            s[what] = torch.tensor(values, dtype=typ, device="cuda") if any(v != off for v in values) else None
        s["x"] = x
        if case["kind"] == "probs":
            return s | {"out": torch.empty_like(x)}
        return s | {"u": torch.rand(R, case["draws"], generator=gen, device="cuda"),
                    "token": torch.full((R, case["draws"]), -1, dtype=torch.int32, device="cuda"),
                    "logprob": torch.zeros(R, case["draws"], device="cuda")}
    layout = _layout(case, int(seed))
    tables, pages = _tables(case, layout, rng)
    start = [0]
    for *_, rows in layout:
        start.append(start[-1] + rows)
    length = [held + tail for _, _, held, tail, _ in layout]
    s |= {"table": _ints(tables), "length": _ints(length), "start": _ints(start), "total": start[-1], "most": max(r for *_, r in layout),
          "lengths": length, "starts": start, "pages": pages, "parent": None, "link": torch.zeros(len(layout), dtype=torch.int32, device="cuda"),
          "shared": torch.zeros(len(layout), dtype=torch.int32, device="cuda")}
    if case["kind"] == "prefixes":
        # what the pages hold is not looked at
        s["k"] = s["v"] = torch.zeros(1, pages, 1, case["page"], case["dim"], dtype=DTYPES[case["type"]], device="cuda")
        return s
    if case["tree"]:
        up = []
        for *_, n in layout:
            up += [-1] + [i - 1 if rng.random() < 0.5 else rng.randint(max(0, i - 5), i - 1) for i in range(1, n)]
        s["parents"], s["parent"] = up, _ints(up)
    s["seen"] = [_lines(s, b).cuda() for b in range(len(layout))]
    shape = (case["layers"], pages, case["kv_heads"], case["page"], case["dim"])
    for name in ("k", "v"):
        s[name] = torch.empty(shape, dtype=DTYPES[case["type"]], device="cuda")
        for i in range(case["layers"]):
            s[name][i].normal_(generator=gen)
    s["q"] = torch.randn(case["layers"], s["total"], case["q_heads"], case["dim"], generator=gen, device="cuda")
    s["out"] = torch.empty_like(s["q"])
    return s


# ---------------- the framework's calls ----------------

def _plan(s):
    """Descriptors and workspaces, which a program keeps with its buffers."""
    if "plan" in s:
        return s["plan"]
    import ctypes
    from nebula_amd import qg
    c, plan, lib = s["case"], {}, qg.lib()

    def ptr(name):
        return s[name].data_ptr() if s.get(name) is not None else None

    def space(name, n):
        plan[name + "_bytes"], plan[name + "_"] = n, torch.empty(max(16, n), dtype=torch.uint8, device="cuda")
        plan[name] = plan[name + "_"].data_ptr()
    if c["kind"] in ("sample", "probs"):
        plan["sampling_"] = qg.Sampling(temperature=ptr("temperature"), top_k=ptr("top_k"), top_p=ptr("top_p"), min_p=ptr("min_p"))
        plan["sampling"] = ctypes.byref(plan["sampling_"])
        space("ws", lib.qg_sample_workspace_bytes(c["rows"], c["cols"]))
    else:
        plan["batch_"] = qg.KvBatch(rows=s["total"], max_rows=s["most"], start=ptr("start"), parent=ptr("parent"))
        plan["cache_"] = qg.KvCache(k=ptr("k"), v=ptr("v"), type=c["type"], layers=c["layers"], pages=s["pages"], kv_heads=c["kv_heads"],
                                    page_tokens=c["page"], head_dim=c["dim"], refs=None, table=ptr("table"), length=ptr("length"),
                                    sequences=s["length"].numel(), table_pages=s["table"].shape[1])
        plan["batch"], plan["cache"] = ctypes.byref(plan["batch_"]), ctypes.byref(plan["cache_"])
        space("prefix", lib.qg_kv_prefixes_bytes(plan["cache"], plan["batch"]))
        if c["kind"] == "shared":
            space("ws", lib.qg_prefix_attention_workspace_bytes(plan["cache"], plan["batch"], c["q_heads"]))
    s["plan"] = plan
    return plan


def _own(s):
    from nebula_amd import qg
    c, p = s["case"], _plan(s)
    if c["kind"] == "sample":
        qg.call("sample", s["token"].data_ptr(), s["logprob"].data_ptr(), s["x"].data_ptr(), c["rows"], c["cols"], c["draws"], p["sampling"],
                s["u"].data_ptr(), p["ws"], p["ws_bytes"])
    elif c["kind"] == "probs":
        qg.call("sampling_softmax", s["out"].data_ptr(), s["x"].data_ptr(), c["rows"], c["cols"], p["sampling"], p["ws"], p["ws_bytes"])
    else:
        qg.call("kv_prefixes", s["link"].data_ptr(), s["shared"].data_ptr(), p["cache"], p["batch"], p["prefix"], p["prefix_bytes"])
        if c["kind"] == "shared":
            for layer in range(c["layers"]):
                qg.call("prefix_attention", s["out"][layer].data_ptr(), s["q"][layer].data_ptr(), c["q_heads"], c["dim"] ** -0.5, p["cache"],
                        layer, p["batch"], p["prefix"], p["prefix_bytes"], p["ws"], p["ws_bytes"])


# ---------------- the plain forms ----------------

def _plain_prefixes(s):
    table, P = s["table"], s["case"]["page"]
    S, W = table.shape
    whole = (s["length"] // P).long()  # full pages of cached tokens
    i, j = torch.arange(S, device="cuda"), torch.arange(W, device="cuda")
    has = s["start"][1:] > s["start"][:-1]
    for a in range(0, S, 64):
        b = slice(a, min(a + 64, S))
        same = (table[b, None] == table[None]) & (table[b, None] >= 0) & (j < torch.minimum(whole[b, None], whole[None])[:, :, None])
        n = same.to(torch.int8).cumprod(-1, dtype=torch.int8).sum(-1)
        n = n.masked_fill((i >= i[b, None]) | ~has | ~has[b, None], 0)
        most = n.amax(-1)
        first = (n == most[:, None]).int().argmax(-1)
        s["shared"][b] = (most * P).int()
        s["link"][b] = torch.where(most > 0, first, -1).int()


def _lines(s, b):
    """[n, n] which rows of sequence b each of its rows descends from, itself included."""
    first, n = s["starts"][b], s["starts"][b + 1] - s["starts"][b]
    seen = torch.ones(n, n, dtype=torch.bool).tril()
    if s["parent"] is not None:
        seen = torch.eye(n, dtype=torch.bool)
        for i in range(n):
            if s["parents"][first + i] >= 0:
                seen[i] |= seen[s["parents"][first + i]]
    return seen


def _plain_shared(s):
    c = s["case"]
    Hkv, D, P, G = c["kv_heads"], c["dim"], c["page"], c["q_heads"] // c["kv_heads"]
    for layer in range(c["layers"]):
        for b, length in enumerate(s["lengths"]):
            first, n = s["starts"][b], s["starts"][b + 1] - s["starts"][b]
            keys = length + n
            pages = s["table"][b, :-(-keys // P)].long()
            K, V = (pool[layer, pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :keys].float() for pool in (s["k"], s["v"]))
            q = s["q"][layer, first:first + n].reshape(n, Hkv, G, D).transpose(0, 1).reshape(Hkv, n * G, D)
            z = (q @ K.transpose(-1, -2)).mul_(D ** -0.5).view(Hkv, n, G, keys)
            z[..., length:].masked_fill_(~s["seen"][b][:, None], -math.inf)
            w = z.sub_(z.amax(-1, keepdim=True)).exp_()
            o = (w.view(Hkv, n * G, keys) @ V) / w.view(Hkv, n * G, keys).sum(-1, keepdim=True)
            s["out"][layer, first:first + n] = o.view(Hkv, n, G, D).transpose(0, 1).reshape(n, -1, D)


def _column(s, what, b, off):
    return s[what][b, None] if s[what] is not None else off


def _kept(s, b):
    """Rows b: the weights that stay, in 64 bits and the tokens' order (0: dropped)."""
    x = s["x"][b]
    T = _column(s, "temperature", b, torch.ones(1, device="cuda")).double()
    k, p, least = _column(s, "top_k", b, 0), _column(s, "top_p", b, 1.0), _column(s, "min_p", b, 0.0)
    best, order = torch.sort(x, dim=-1, descending=True, stable=True)
    place = torch.arange(x.shape[1], device="cuda")
    w = torch.exp((best.double() - best[:, :1].double()) / torch.where(T > 0, T, 1.0))
    w = torch.where(T > 0, w, (place == 0).double())
    if s["top_k"] is not None:
        w = torch.where((k > 0) & (place >= k), 0.0, w)
    if s["top_p"] is not None:
        upto = w.cumsum(-1)
        before = torch.nn.functional.pad(upto[:, :-1], (1, 0))
        w = torch.where((p < 1) & (place > 0) & (before >= p.double() * upto[:, -1:]), 0.0, w)
    if s["min_p"] is not None:
        w = torch.where(w >= least.double(), w, 0.0)
    return torch.empty_like(w).scatter_(1, order, w)


def _blocks(case):
    n = max(1, (1 << 24) // case["cols"])
    return [slice(i, min(i + n, case["rows"])) for i in range(0, case["rows"], n)]


def _plain_sample(s):
    for b in _blocks(s["case"]):
        w = _kept(s, b)
        upto = w.cumsum(-1)
        goal = s["u"][b].double() * upto[:, -1:]
        last = w.shape[1] - 1 - (w > 0).flip(-1).int().argmax(-1, keepdim=True)
        pick = torch.minimum(torch.searchsorted(upto, goal, right=True), last)
        s["token"][b] = pick.int()
        s["logprob"][b] = torch.log(w.gather(1, pick) / upto[:, -1:]).float()


def _plain_probs(s):
    for b in _blocks(s["case"]):
        w = _kept(s, b)
        s["out"][b] = (w / w.sum(-1, keepdim=True)).float()


def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        _own(s)
    else:
        {"prefixes": _plain_prefixes, "shared": _plain_shared, "sample": _plain_sample, "probs": _plain_probs}[kind](s)
    if kind == "prefixes":
        return {"link": s["link"], "shared": s["shared"]}
    if kind == "sample":
        return {"token": s["token"], "logprob": s["logprob"]}
    return s["out"]


# ---------------- what a pass needs, and its exact result ----------------

def work(case):
    if case["kind"] in ("sample", "probs"):
        n = case["rows"] * case["cols"]
        return {"bytes": 8 * n if case["kind"] == "probs" else 4 * n + 12 * case["rows"] * case["draws"], "flops": 4 * n}
    layout, P = _layout(case), case["page"]
    S = len(layout)
    if case["kind"] == "prefixes":
        return {"bytes": 4 * sum((held + tail) // P for _, _, held, tail, _ in layout) + 4 * (4 * S + 1), "flops": 0}
    # each page of the system text and the prompts once, as far as a sequence holds it
    most = {}
    for p, _, held, *_ in layout:
        most[p] = max(most.get(p, 0), held // P)
    shared = sum(max(0, n - case["system"] // P) for n in most.values()) + min(case["system"] // P, max(most.values()))
    tokens = shared * P + sum(held % P + tail + rows for _, _, held, tail, rows in layout)
    pairs = sum(rows * (held + tail) + rows * (rows + 1) // 2 for _, _, held, tail, rows in layout)
    rows, D, Hq, L = sum(r for *_, r in layout), case["dim"], case["q_heads"], case["layers"]
    return {"bytes": L * (tokens * case["kv_heads"] * D * 2 * SIZE[case["type"]] + rows * Hq * D * 8), "flops": L * 4 * pairs * Hq * D}


def exact(case, seed):
    if case["kind"] == "prefixes":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "shared":
        return _exact_shared(s)
    tokens, logs, probs = [], [], []
    for r in range(case["rows"]):
        x = s["x"][r].double()
        T, k, p, least = (float(s[n][r]) if s[n] is not None else d for n, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
        if T == 0:
            first = int((s["x"][r] == s["x"][r].max()).nonzero()[0])
            q = torch.zeros_like(x)
            q[first] = 1
        else:
            q = torch.softmax(x / T, 0)
            stays = q.new_ones(q.shape, dtype=torch.bool)
            if 0 < k < x.numel():
                kth = torch.topk(x, int(k)).values[-1]
                stays = x > kth
                level = (x == kth).nonzero()[:, 0]
                stays[level[:int(k) - int(stays.sum())]] = True
            q = q * stays
            if p < 1:  # walk down the distinct values, then through the equal ones in order
                q = q / q.sum()
                values, inverse = torch.unique(x, return_inverse=True)
                mass = torch.zeros(values.numel(), dtype=torch.float64, device="cuda").index_add_(0, inverse, q)
                above = mass.flip(0).cumsum(0).flip(0) - mass
                border = int((above < p).nonzero()[0])
                level = ((inverse == border) & (q > 0)).nonzero()[:, 0]
                each = float(q[level[0]]) if level.numel() else 1.0
                n = max(1, math.ceil((p - float(above[border])) / each - 1e-12))
                stays = (inverse > border) & stays
                stays[level[:n]] = True
                q = q * stays
            q = torch.where(q >= least * q.max(), q, 0.0)
            q = q / q.sum()
        if case["kind"] == "probs":
            probs.append(q)
            continue
        upto = q.cumsum(0)
        at = (upto <= s["u"][r].double()[:, None] * upto[-1]).sum(-1).clamp_max(int(q.nonzero()[-1]))
        tokens.append(at.int())
        logs.append(torch.log(q[at]))
    if case["kind"] == "probs":
        return torch.stack(probs)
    return {"token": torch.stack(tokens), "logprob": torch.stack(logs)}


def _exact_shared(s):
    case = s["case"]
    Hkv, G, D, P = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lengths"]):
        first, n = s["starts"][b], s["starts"][b + 1] - s["starts"][b]
        t = torch.arange(length + n, device="cuda")
        page, slot = s["table"][b].long()[t // P], t % P
        hidden = torch.zeros(n, length + n, dtype=torch.bool)
        for i in range(n):
            hidden[i, length:] = True
            j = i
            while j >= 0:
                hidden[i, length + j] = False
                j = s["parents"][first + j] if s["parent"] is not None else j - 1
        hidden = hidden.cuda()
        for layer in range(case["layers"]):
            for h in range(Hkv):
                K, V = s["k"][layer, page, h, slot].double(), s["v"][layer, page, h, slot].double()
                for g in range(h * G, (h + 1) * G):
                    z = s["q"][layer, first:first + n, g].double() @ K.T / math.sqrt(D)
                    out[layer, first:first + n, g] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ V
    return out
