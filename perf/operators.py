"""The serving operators of this package as measurable cases: attention of a decode batch that shares long prefixes,
packed-row indices and block tables from request lengths, and token sampling.

``run`` computes a case either in its plain form (elementary torch operations) or, with ``own`` set, through the
package's public entry points.  ``exact`` restates the definitions in 64 bits.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"


def _package():
    """The package of the tree that this file lies in."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "falcon-perception_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from fpkv import paged_attention, sampling
    return paged_attention, sampling


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # four short questions about one small picture: every launch counts, the data fits in a few caches
        {"name": "shared 4x512", "op": "shared", "groups": 1, "rows": 4, "prefix": 512, "suffix": 64,
         "hq": 16, "hkv": 8, "d": 128, "dtype": "bf16", "spare": 0},
        # the ordinary batch: 64 requests about one long document, answers of up to 512 tokens
        {"name": "shared 64x8192", "op": "shared", "groups": 1, "rows": 64, "prefix": 8192, "suffix": 512,
         "hq": 16, "hkv": 8, "d": 128, "dtype": "bf16", "spare": 0},
        # several pictures of different sizes with different numbers of questions each, some requests that share nothing
        {"name": "shared 7 groups fp16 d64", "op": "shared", "groups": 7, "rows": 13, "prefix": 2944, "suffix": 301,
         "hq": 4, "hkv": 2, "d": 64, "dtype": "fp16", "spare": 5},
        # the largest: 256 requests over one 32K prefix
        {"name": "shared 256x32768", "op": "shared", "groups": 1, "rows": 256, "prefix": 32768, "suffix": 512,
         "hq": 16, "hkv": 8, "d": 128, "dtype": "bf16", "spare": 0},
        # one chat: a single row of logits, nucleus sampling
        {"name": "sample 1x65536", "op": "sample", "rows": 1, "vocab": 65536, "dtype": "bf16", "filters": "p", "masked": 0.0},
        # a decode batch in which every request brings its own settings, some of them greedy
        {"name": "sample 64x65536 mixed", "op": "sample", "rows": 64, "vocab": 65536, "dtype": "bf16", "filters": "mixed",
         "masked": 0.0},
        # an odd vocabulary with forbidden tokens, top-k only
        {"name": "sample 33x49999 topk", "op": "sample", "rows": 33, "vocab": 49999, "dtype": "fp16", "filters": "k",
         "masked": 0.3},
        # the largest: a wide batch of 32-bit logits
        {"name": "sample 512x131072 fp32", "op": "sample", "rows": 512, "vocab": 131072, "dtype": "fp32", "filters": "mixed",
         "masked": 0.0},
        # a step that admits three short prompts
        {"name": "tables 3", "op": "tables", "requests": 3, "longest": 200, "start": 0, "align": 128, "slack": 0},
        # a mixed step: chunks of prompts in flight next to one-token rows
        {"name": "tables 64", "op": "tables", "requests": 64, "longest": 512, "start": 8192, "align": 128, "slack": 777},
        # the largest: whole prompts of up to 4K tokens for 512 requests
        {"name": "tables 512", "op": "tables", "requests": 512, "longest": 4096, "start": 4096, "align": 16, "slack": 4096},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shared", "shared", "sample", "sample", "tables"])
    if op == "shared":
        hq, hkv, d = rng.choice([(16, 8, 128), (16, 8, 128), (4, 2, 128), (16, 16, 128), (16, 8, 64), (4, 2, 64), (8, 1, 128),
                                 (16, 4, 128), (6, 2, 128)])
        while True:
            groups = _log_int(rng, 1, 12)
            c = {"op": op, "groups": groups, "rows": _log_int(rng, 2, 256 // groups), "prefix": PAGE * _log_int(rng, 1, 256),
                 "suffix": _log_int(rng, 1, 1024), "hq": hq, "hkv": hkv, "d": d, "dtype": rng.choice(["bf16", "bf16", "fp16"]),
                 "spare": rng.choice([0, 0, 1, 5])}
            rows = groups * c["prefix"] + (groups * c["rows"] + c["spare"]) * (c["suffix"] + PAGE)
            # scores of the plain form, and the pool, stay below those of the largest listed case
            if (groups * c["rows"] + c["spare"]) * hq * rows <= 256 * 16 * 164000 and rows * hkv * d <= 164000 * 8 * 128:
                return c
    if op == "sample":
        while True:
            c = {"op": op, "rows": _log_int(rng, 1, 512), "vocab": _log_int(rng, 32, 262144),
                 "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "filters": rng.choice(["p", "k", "mixed", "mixed", "none"]),
                 "masked": rng.choice([0.0, 0.0, 0.3])}
            if c["rows"] * c["vocab"] <= 512 * 131072:
                return c
    while True:
        c = {"op": op, "requests": _log_int(rng, 1, 512), "longest": _log_int(rng, 1, 4096), "start": rng.choice([0, 1, 4096, 8191]),
             "align": rng.choice([1, 16, 128]), "slack": rng.choice([0, 1, 500])}
        if c["requests"] * (c["longest"] + c["start"]) <= 512 * 8192:
            return c


# ---------------------------------------------------------- attention, shared prefixes
def _shared_layout(case, seed):
    """Group sizes, prefix lengths and suffix lengths (host).  A single group has exactly the sizes named; with several
    the sizes run from half of them to all of them, dealt out by the seed (the batch size is the case's own)."""
    rng = np.random.default_rng(seed)
    G = case["groups"]
    if G == 1:
        rows, prefix = [case["rows"]], [case["prefix"]]
    else:
        least, top = max(1, case["rows"] // 2), case["prefix"] // PAGE
        rows = rng.permutation([least + (case["rows"] - least) * g // (G - 1) for g in range(G)]).tolist()
        prefix = [PAGE * int(rng.integers(max(1, top // 2), top + 1)) for _ in range(G)]
    n = sum(rows) + case["spare"]
    suffix = rng.integers(1, case["suffix"] + 1, size=n).tolist()
    return rows, prefix, suffix, rng


def _prepare_shared(case, seed):
    rows, prefix, suffix, rng = _shared_layout(case, seed)
    dtype, hkv, hq, d = DTYPES[case["dtype"]], case["hkv"], case["hq"], case["d"]
    B = sum(rows) + case["spare"]
    suffix_pages = [(s + PAGE - 1) // PAGE for s in suffix]
    group_of = [g for g, r in enumerate(rows) for _ in range(r)] + [-1] * case["spare"]
    n_pages = 1 + sum(prefix) // PAGE + sum(suffix_pages) + 8
    order = (rng.permutation(n_pages - 1) + 1).tolist()
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    if own:
        fpkv, _ = _package()
        cache = fpkv.PagedKVCache(n_pages, PAGE, B + 1, hkv, d, 1, dtype, DEVICE)
        cache.free_pages = order
        slots, first = [], {}
        for b, g in enumerate(group_of):
            if g < 0 or g not in first:
                slot = cache.allocate()
                cache.reserve(slot, None, (prefix[g] if g >= 0 else 0) + suffix[b])
                first.setdefault(g, slot)
            else:
                slot = cache.share_prefix(first[g], prefix[g])
                cache.reserve(slot, None, prefix[g] + suffix[b])
            slots.append(slot)
        pages = [list(cache.page_table_cpu[s]) for s in slots]
        pool = cache.kv_cache[0, :, 0]
        state = {"cache": cache, "shared": cache.prefix_groups(slots)}
    else:
        free, pages, first = list(order), [], {}

        def take(n):
            got = free[-n:]
            del free[-n:]
            return got
        for b, g in enumerate(group_of):
            if g >= 0:
                if g not in first:
                    first[g] = take(prefix[g] // PAGE)
                pages.append(first[g] + take(suffix_pages[b]))
            else:
                pages.append(take(suffix_pages[b]))
        slots = list(range(1, B + 1))
        pool = torch.zeros(2, hkv, n_pages * PAGE, d, dtype=dtype, device=DEVICE)
        table = torch.full((B + 1, n_pages), -1, dtype=torch.int64)
        for s, p in zip(slots, pages):
            table[s, torch.tensor(p)] = torch.arange(len(p))
        state = {"pool": pool, "physical_to_logical": table.to(DEVICE)}

    # contents in logical order -- the prefixes, then every row's own pages -- scattered to wherever the pages are
    where, seen = [], set()
    for b, g in enumerate(group_of):
        own_from = prefix[g] // PAGE if g >= 0 else 0
        if g >= 0 and g not in seen:
            seen.add(g)
            where += pages[b][:own_from]
        where += pages[b][own_from:]
    at = (torch.tensor(where, device=DEVICE)[:, None] * PAGE + torch.arange(PAGE, device=DEVICE)).reshape(-1)
    for kv in range(2):
        for h in range(hkv):
            pool[kv, h, at] = torch.randn(at.numel(), d, generator=gen, device=DEVICE).to(dtype)
    state["q"] = torch.randn(B, hq, 1, d, generator=gen, device=DEVICE).to(dtype)
    state["batch_idx"] = torch.tensor(slots, device=DEVICE)
    last = [(prefix[g] if g >= 0 else 0) + s - 1 for g, s in zip(group_of, suffix)]
    state["input_pos"] = torch.tensor(last, dtype=torch.int32, device=DEVICE)
    return state


def _run_shared(state):
    if own:
        return state["cache"].decode_attention(0, state["q"], state["batch_idx"], state["input_pos"], shared=state["shared"])
    # every query against every row of the pool; what a row may see is decided by its inverse page table
    pool, q, pos = state["pool"], state["q"], state["input_pos"].long()
    _, H, R, D = pool.shape
    B, Hq = q.shape[:2]
    page = state["physical_to_logical"][state["batch_idx"]]                                   # (B, n_pages)
    logical = (page[:, :, None] * PAGE + torch.arange(PAGE, device=q.device)).reshape(B, R)
    seen = (logical >= 0) & (logical <= pos[:, None])
    qh = q.float().view(B, H, Hq // H, D).transpose(0, 1).reshape(H, -1, D)                    # (H, B * rep, D)
    s = torch.matmul(qh, pool[0].float().transpose(1, 2)).view(H, B, Hq // H, R) * (D ** -0.5)
    s.masked_fill_(~seen[None, :, None, :], float("-inf"))
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - m)
    l = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(H, -1, R), pool[1].float()).view(H, B, Hq // H, D) / l
    out = o.transpose(0, 1).reshape(B, Hq, 1, D).to(q.dtype)
    lse = (m + torch.log(l)).transpose(0, 1).reshape(B, Hq, 1)
    return out, lse


def _exact_shared(case, seed):
    """Row by row in 64 bits over the row's own keys in order."""
    rows, prefix, suffix, _ = _shared_layout(case, seed)
    state = _prepare_shared(case, seed)
    q = state["q"].double()
    pos = state["input_pos"].tolist()
    if "pool" in state:
        pool, p2l = state["pool"], state["physical_to_logical"]
    else:
        pool, p2l = state["cache"].kv_cache[0, :, 0], state["cache"].physical_to_logical
    rep = case["hq"] // case["hkv"]
    outs, lses = [], []
    for b in range(q.shape[0]):
        logical = p2l[state["batch_idx"][b]]
        mine = torch.nonzero(logical >= 0).flatten()
        mine = mine[torch.argsort(logical[mine])]
        at = (mine[:, None] * PAGE + torch.arange(PAGE, device=mine.device)).reshape(-1)[:pos[b] + 1]
        k, v = pool[0][:, at].double(), pool[1][:, at].double()
        s = torch.einsum("hrd,hkd->hrk", q[b, :, 0].view(case["hkv"], rep, -1), k) / math.sqrt(case["d"])
        lse = torch.logsumexp(s, -1)
        outs.append(torch.einsum("hrk,hkd->hrd", torch.exp(s - lse[..., None]), v).reshape(case["hq"], 1, -1))
        lses.append(lse.reshape(case["hq"], 1))
    return torch.stack(outs), torch.stack(lses)


def _work_shared(case):
    # sizes in expectation where they are drawn: a prefix is read once a group, every row's own keys once
    G, spread = case["groups"], 1.0 if case["groups"] == 1 else 0.75
    rows, prefix = case["rows"] * spread, case["prefix"] * spread
    B, own_keys = G * rows + case["spare"], (case["suffix"] + 1) / 2
    es = DTYPES[case["dtype"]].itemsize
    keys = G * prefix + B * own_keys
    pairs = G * rows * prefix + B * own_keys
    return {"bytes": keys * 2 * case["hkv"] * case["d"] * es + B * case["hq"] * (2 * case["d"] * es + 4),
            "flops": 4.0 * pairs * case["hq"] * case["d"]}


# ------------------------------------------------------------------ sampling
def _prepare_sample(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    B, V, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    # a broad tail with a handful of likely tokens in every row, as a language model's last layer gives them
    x = torch.randn(B, V, generator=gen, device=DEVICE) * 2.5
    likely = torch.randint(0, V, (B, 12), generator=gen, device=DEVICE)
    x.scatter_add_(1, likely, 6 + 3 * torch.randn(B, 12, generator=gen, device=DEVICE))
    if case["masked"]:
        x.masked_fill_(torch.rand(B, V, generator=gen, device=DEVICE) < case["masked"], float("-inf"))
        x[:, 0] = 0.0                                   # a token that is always allowed
    u = torch.rand(4, B, generator=gen, device=DEVICE)
    s = {"logits": x.to(dtype), "uniform": u[0].contiguous(), "temperature": 0.5 + u[1], "top_k": None, "top_p": None, "min_p": None}
    kind = case["filters"]
    if kind in ("k", "mixed"):
        s["top_k"] = (1 + 200 * u[2]).to(torch.int32)
    if kind in ("p", "mixed"):
        s["top_p"] = 0.6 + 0.4 * u[3]
    if kind == "mixed":
        i = torch.arange(B, device=DEVICE)
        s["min_p"] = torch.where(i % 4 == 3, 0.1 * u[2], torch.zeros_like(u[2]))
        s["top_k"] = torch.where(i % 4 == 1, s["top_k"], torch.zeros_like(s["top_k"]))          # 0: no limit
        s["top_p"] = torch.where(i % 4 == 0, torch.ones_like(s["top_p"]), s["top_p"])          # 1: no limit
        s["temperature"] = torch.where(i % 8 == 7, torch.zeros_like(u[1]), s["temperature"])    # 0: greedy
    return s


def _run_sample(state):
    if own:
        _, sampling = _package()
        return sampling.sample(state["logits"], state["uniform"], temperature=state["temperature"], top_k=state["top_k"],
                               top_p=state["top_p"], min_p=state["min_p"])
    x = state["logits"].double()
    B, V = x.shape
    t = state["temperature"].double()[:, None]
    k = state["top_k"].long()[:, None] if state["top_k"] is not None else torch.zeros(B, 1, dtype=torch.long, device=x.device)
    p = state["top_p"].double()[:, None] if state["top_p"] is not None else torch.ones(B, 1, dtype=torch.double, device=x.device)
    low = state["min_p"].double()[:, None] if state["min_p"] is not None else torch.zeros(B, 1, dtype=torch.double, device=x.device)
    greedy = t <= 0
    v, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((v - v[:, :1]) / torch.where(greedy, torch.ones_like(t), t))
    rank = torch.arange(V, device=x.device)[None]
    kept = (v > float("-inf")) & ((k <= 0) | (rank < k)) & (~greedy | (rank == 0))
    w = torch.where(kept, w, torch.zeros_like(w))
    mass = torch.cumsum(w, 1)
    kept &= (p >= 1) | (mass - w < p * mass[:, -1:]) | (rank == 0)
    kept &= w >= low
    w = torch.where(kept, w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, order, w)                                              # back in the order of the vocabulary
    mass = torch.cumsum(w, 1)
    total = mass[:, -1:]
    token = (mass <= state["uniform"].double()[:, None] * total).sum(1, keepdim=True)
    logprob = torch.log(w.gather(1, token.clamp(max=V - 1)) / total)
    return token[:, 0], logprob[:, 0].float()


def _exact_sample(case, seed):
    s = _prepare_sample(case, seed)
    logits = s["logits"].double().cpu().numpy()
    par = {n: (s[n].double().cpu().numpy() if s[n] is not None else None) for n in ("uniform", "temperature", "top_k", "top_p", "min_p")}
    tokens, logprobs = [], []
    for b, x in enumerate(logits):
        T = par["temperature"][b]
        if T <= 0:
            tokens.append(int(np.argmax(x)))
            logprobs.append(0.0)
            continue
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -np.inf]
        if par["top_k"] is not None and par["top_k"][b] > 0:
            order = order[:int(par["top_k"][b])]
        w = np.exp((x[order] - x[order[0]]) / T)
        n = len(order)
        if par["top_p"] is not None and par["top_p"][b] < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            n = max(1, int(np.count_nonzero(before < par["top_p"][b] * w.sum())))
        if par["min_p"] is not None:
            n = min(n, int(np.count_nonzero(w >= par["min_p"][b])))
        ids = np.sort(order[:n])
        w = np.exp((x[ids] - x[order[0]]) / T)
        c = np.cumsum(w)
        j = min(int(np.searchsorted(c, par["uniform"][b] * c[-1], side="right")), n - 1)
        tokens.append(int(ids[j]))
        logprobs.append(float(np.log(w[j] / c[-1])))
    return torch.tensor(tokens), torch.tensor(logprobs, dtype=torch.double)


def _work_sample(case):
    B, V = case["rows"], case["vocab"]
    # one look at every logit for the maximum, one exponential and one sum
    return {"bytes": B * V * DTYPES[case["dtype"]].itemsize + B * 32, "flops": 4.0 * B * V}


# --------------------------------------------------------- indices of a step
def _tables_layout(case, seed):
    """Lengths evenly spread from one token to the longest, a quarter of them one token (requests that decode), dealt
    out by the seed; where each request starts is drawn."""
    rng = np.random.default_rng(seed)
    N = case["requests"]
    i = np.arange(N)
    lens = rng.permutation(np.where(i % 4 == 3, 1, 1 + (case["longest"] - 1) * (N - i) // N))
    starts = rng.integers(0, case["start"] + 1, size=N)
    row = int((-(-lens // case["align"]) * case["align"]).sum()) + case["slack"]
    return lens, starts, row, rng


def _prepare_tables(case, seed):
    lens, starts, row, rng = _tables_layout(case, seed)
    N = case["requests"]
    need = [int(-(-(a + n) // PAGE)) for a, n in zip(starts, lens)]
    n_pages = 1 + sum(need)
    order = (rng.permutation(n_pages - 1) + 1).tolist()
    width = (case["start"] + case["longest"] + PAGE - 1) // PAGE
    if own:
        fpkv, _ = _package()
        cache = fpkv.PagedKVCache(n_pages, PAGE, N + 1, 1, 64, 1, torch.bfloat16, DEVICE)
        cache.free_pages = order
        slots = []
        for a, n in zip(starts, lens):
            slots.append(cache.allocate())
            cache.reserve(slots[-1], None, int(a + n))
        cache.flush_tables()
        state = {"cache": cache}
    else:
        free, slots = list(order), list(range(1, N + 1))
        table = torch.full((N + 1, n_pages), -1, dtype=torch.int64)
        table[0] = 0
        for s, n in zip(slots, need):
            table[s, :n] = torch.tensor(free[-n:])
            del free[-n:]
        state = {"page_table": table.to(DEVICE)}
    state["slots"] = torch.tensor(slots, device=DEVICE)
    state["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
    state["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEVICE)
    state["tokens"] = torch.tensor(rng.integers(1, 65536, size=int(lens.sum())), device=DEVICE)
    state.update(row=row, width=width, align=case["align"])
    return state


def _run_tables(state):
    if own:
        t = state["cache"].step_tables(state["slots"], state["starts"], state["lens"], row_tokens=state["row"],
                                       width=state["width"], align=state["align"], tokens=state["tokens"])
        return [t.input_ids, t.input_pos, t.batch_idx, t.pool_row, t.block_table, t.seq_lens, t.offsets, t.last]
    pt, slots, starts, lens = state["page_table"], state["slots"], state["starts"].long(), state["lens"].long()
    a = state["align"]
    ends = torch.cumsum((lens + a - 1) // a * a, 0)
    first = ends - (lens + a - 1) // a * a
    before = torch.cumsum(lens, 0) - lens
    t = torch.arange(state["row"], device=pt.device)
    r = torch.searchsorted(ends, t, right=True).clamp(max=slots.numel() - 1)
    i = t - first[r]
    live = i < lens[r]
    pos = torch.where(live, starts[r] + i, torch.zeros_like(i))
    bidx = torch.where(live, slots[r], torch.zeros_like(r))
    ids = torch.where(live, state["tokens"][torch.where(live, before[r] + i, torch.zeros_like(i))], torch.zeros_like(r))
    page = pt[bidx, pos // PAGE]
    pool_row = torch.where(live & (page >= 0), page * PAGE + pos % PAGE, torch.full_like(page, -1))
    total = starts + lens
    j = torch.arange(state["width"], device=pt.device)
    inside = j[None] * PAGE < total[:, None]
    block = torch.where(inside, pt[slots][:, j.clamp(max=pt.shape[1] - 1)], torch.full_like(inside, -1, dtype=torch.int64)).int()
    offsets = torch.cat([first, ends[-1:]]).int()
    return [ids[None], pos[None], bidx[None], pool_row, block, total.int(), offsets, (first + lens - 1).int()]


def _work_tables(case):
    N, mean = case["requests"], 0.75 * (case["longest"] + 1) / 2 + 0.25
    row = N * (mean + (case["align"] - 1) / 2) + case["slack"]
    pages = N * (mean + case["start"] / 2) / PAGE + N / 2
    width = (case["start"] + case["longest"] + PAGE - 1) // PAGE
    return {"bytes": N * mean * 8 + row * 32 + pages * 8 + N * width * 4 + N * 28, "flops": 8.0 * row}


# -------------------------------------------------------------------- the calls
def prepare(case, seed):
    return {"op": case["op"], **{"shared": _prepare_shared, "sample": _prepare_sample, "tables": _prepare_tables}[case["op"]](case, seed)}


def run(state):
    return {"shared": _run_shared, "sample": _run_sample, "tables": _run_tables}[state["op"]](state)


def exact(case, seed):
    if case["op"] == "tables":
        return None
    return {"shared": _exact_shared, "sample": _exact_sample}[case["op"]](case, seed)


def work(case):
    return {"shared": _work_shared, "sample": _work_sample, "tables": _work_tables}[case["op"]](case)
