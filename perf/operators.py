"""Work of the prompt and single-token serving path, measured operator by operator.

Four operators, each with its plain form in elementary torch operations and the
call a user makes of this package (``own`` selects which):

* ``prompt``: causal grouped-query attention over whole packed prompts
  (``respect_b200.kernels.attention.prompt_attention``).
* ``paged``: attention of one new token per sequence over a paged KV cache
  (``respect_b200.kernels.attention.paged_attention``).
* ``pages``: what happens to the pages of that cache between two forwards:
  forking samples off a prompt, and a round of drafted tokens of which an
  accepted path stays (``respect_b200.decoding.kv_pages.PagedKVCache``).
* ``logprobs``: log probability of one given token per row, the row's entropy
  and its best alternatives (``respect_b200.decoding.acceptance.token_logprobs``).
"""
import math

import torch

own = False

D = 128
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
VOCAB = 152064


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one short system prompt alone: the latency of a whole call counts
        dict(name="prompt_short", op="prompt", dtype="bf16", H=28, HK=4, lens="96"),
        # the prompts of 16 frame streams in one call, near 4,096 tokens each
        dict(name="prompt_streams", op="prompt", dtype="bf16", H=28, HK=4,
             lens="4096 4033 4096 3891 4210 4096 3686 4096 4100 4095 4096 4301 4096 3999 4096 4127"),
        # one long document, grouped by four
        dict(name="prompt_long", op="prompt", dtype="bf16", H=32, HK=8, lens="32768"),
        # the fp32 path that parity runs use; ragged, with an empty and a one-token prompt
        dict(name="prompt_f32", op="prompt", dtype="f32", H=28, HK=4, lens="1536 700 0 1 333"),
        # one frame stream decoding: few rows over one cache, split over its length
        dict(name="paged_one", op="paged", dtype="bf16", H=28, HK=4, page=16, lens="4133"),
        # a serving batch of 64 sequences of mixed lengths
        dict(name="paged_batch", op="paged", dtype="bf16", H=32, HK=8, page=64,
             lens=" ".join(str(512 + (i * 2711) % 11519) for i in range(64))),
        # fp32 cache, odd page size, an empty sequence
        dict(name="paged_f32", op="paged", dtype="f32", H=28, HK=4, page=24, lens="1583 0 300 2047 1 5120"),
        # samples forked off two cached prompts, with the first token of each written
        dict(name="pages_fork", op="pages_fork", dtype="bf16", L=28, HK=4, page=16, lens="703 1000", each=8),
        # a verification round of four streams: 256 drafted nodes each, accepted paths of up to 32
        dict(name="pages_round", op="pages_round", dtype="bf16", L=28, HK=4, page=16, lens="400 433 371 512",
             nodes=256, accept="32 7 1 19"),
        # one decoded token
        dict(name="logprobs_one", op="logprobs", dtype="f32", rows=1, V=VOCAB, top=5, offset=0, size=0),
        # every node of a 128-node trie, the action tokens excluded
        dict(name="logprobs_trie", op="logprobs", dtype="f32", rows=128, V=VOCAB, top=20, offset=151700, size=300),
        # scoring of a prompt, bf16 logits, no alternatives
        dict(name="logprobs_prompt", op="logprobs", dtype="bf16", rows=2000, V=VOCAB, top=0, offset=0, size=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "paged", "paged", "pages_fork", "pages_round", "logprobs", "logprobs"])
    heads = rng.choice([(28, 4), (32, 8), (4, 2), (16, 16), (8, 1), (12, 4), (40, 8)])
    if op == "prompt":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        budget = _log_int(rng, 64, 32768 if dtype == "bf16" else 4096)
        lens = []
        for _ in range(rng.randint(1, 16)):
            n = min(budget - sum(lens), _log_int(rng, 1, max(2, budget)))
            lens.append(max(n, 0))
        rng.shuffle(lens)
        return dict(op=op, dtype=dtype, H=heads[0], HK=heads[1], lens=" ".join(map(str, lens)))
    if op == "paged":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        budget = _log_int(rng, 64, 300000 if dtype == "bf16" else 40000)
        lens = []
        for _ in range(_log_int(rng, 1, 128)):
            n = min(budget - sum(lens), _log_int(rng, 1, max(2, budget)))
            lens.append(max(n, 0))
        rng.shuffle(lens)
        return dict(op=op, dtype=dtype, H=heads[0], HK=heads[1], page=rng.choice([8, 16, 24, 32, 64, 100, 128]),
                    lens=" ".join(map(str, lens)))
    if op.startswith("pages"):
        L, page = _log_int(rng, 1, 28), rng.choice([8, 16, 24, 32, 64])
        HK = heads[1]
        tokens = 400000 // (L * HK) // (2 if rng.random() < 0.5 else 1)   # of about 0.2 GB of cache
        c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), L=L, HK=HK, page=page)
        n = rng.randint(1, 4)
        lens = [_log_int(rng, 1, max(2, tokens // (2 * n))) for _ in range(n)]
        c["lens"] = " ".join(map(str, lens))
        if op == "pages_fork":
            c["each"] = rng.randint(1, 8)
        else:
            c["nodes"] = min(rng.choice([8, 33, 64, 128, 256]), max(1, tokens // (4 * n)))
            c["accept"] = " ".join(str(rng.randint(0, min(32, c["nodes"]))) for _ in range(n))
        return c
    dtype = rng.choice(["f32", "f32", "bf16"])
    V = rng.choice([VOCAB, 2048, 32000, _log_int(rng, 40, 200000)])
    rows = _log_int(rng, 1, max(1, min(2000, 304128000 // V // (2 if dtype == "f32" else 1))))
    size = rng.choice([0, V // 50, V // 3])
    return dict(op=op, dtype=dtype, rows=rows, V=V, top=rng.choice([0, 1, 5, 20, 32]),
                offset=rng.randint(0, V - size) if size else 0, size=size)


def _ints(text):
    return [int(x) for x in text.split()]


# ---------------------------------------------------------------- inputs
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _prepare_prompt(c, g):
    """q, k and v as a fused projection leaves them: slices of one [tokens, (H + 2 HK) D] tensor."""
    lens, H, HK = _ints(c["lens"]), c["H"], c["HK"]
    T = sum(lens)
    qkv = torch.randn(max(T, 1), H + 2 * HK, D, device=DEV, generator=g)[:T]
    qkv[:, :H] *= torch.rand(H, 1, device=DEV, generator=g) * 1.5 + 0.5      # heads of different sharpness
    qkv = qkv.to(DTYPES[c["dtype"]])
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return dict(q=qkv[:, :H], k=qkv[:, H:H + HK], v=qkv[:, H + HK:], cu=_i32(cu), lens=lens)


def _page_tables(c, g, lens, spare):
    """Tables of sequences whose pages lie anywhere in the pool; unused entries are -1."""
    ps = c["page"]
    need = [(n + ps - 1) // ps for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, device=DEV, generator=g)[:sum(need)].to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, pages


def _prepare_paged(c, g):
    lens, H, HK, ps = _ints(c["lens"]), c["H"], c["HK"], c["page"]
    dt = DTYPES[c["dtype"]]
    table, pages = _page_tables(c, g, lens, 8)
    kv = torch.empty(2, pages, HK, ps, D, device=DEV, dtype=dt)
    for p in range(0, pages, 1024):     # in pieces: fp32 noise for a whole cache is large
        kv[:, p:p + 1024] = torch.randn(kv[:, p:p + 1024].shape, device=DEV, generator=g).to(dt)
    q = torch.randn(len(lens), H, D, device=DEV, generator=g)
    q *= torch.rand(H, 1, device=DEV, generator=g) * 1.5 + 0.5
    return dict(q=q.to(dt), k=kv[0], v=kv[1], table=table, lengths=_i32(lens), lens=lens)


def _prepare_pages(c, g):
    lens, L, HK, ps = _ints(c["lens"]), c["L"], c["HK"], c["page"]
    dt = DTYPES[c["dtype"]]
    n = len(lens)
    fork = c["op"] == "pages_fork"
    per_seq = (max(lens) + (1 if fork else c["nodes"]) + ps - 1) // ps + 1
    seqs = n + n * c["each"] if fork else n
    spare = n * c["each"] * 2 if fork else n * ((c["nodes"] + ps - 1) // ps + 1)
    table0, pages = _page_tables(c, g, lens, spare)
    st = dict(store=torch.randn(L, 2, pages, HK, ps, D, device=DEV, generator=g).to(dt),
              table=torch.full((seqs, per_seq), -1, dtype=torch.int32, device=DEV),
              lengths=torch.zeros(seqs, dtype=torch.int32, device=DEV),
              held=torch.zeros(seqs, dtype=torch.int32, device=DEV),
              refs=torch.zeros(pages, dtype=torch.int32, device=DEV))
    st["table"][:n, :table0.shape[1]] = table0
    st["lengths"][:n] = _i32(lens)
    st["held"][:n] = _i32([(x + ps - 1) // ps for x in lens])
    st["refs"][table0[table0 >= 0].long()] = 1
    if fork:
        st["src"] = _i32([i for i in range(n) for _ in range(c["each"])])
        st["dst"] = _i32(list(range(n, seqs)))
        st["ones"] = _i32([1] * (seqs - n))
        T = seqs - n
    else:
        accept = _ints(c["accept"])
        paths = torch.zeros(n, max(max(accept), 1), dtype=torch.int32)
        for i, m in enumerate(accept):      # strictly increasing node numbers, as of a path down a trie
            pick = torch.randperm(c["nodes"], device=DEV, generator=g)[:m].sort().values
            paths[i, :m] = pick.to(torch.int32).cpu()
        st["seqs"], st["base"] = _i32(list(range(n))), _i32(lens)
        st["nodes"] = _i32([c["nodes"]] * n)
        st["cu"] = _i32([c["nodes"] * i for i in range(n + 1)])
        st["paths"], st["accept"] = paths.to(DEV), _i32(accept)
        T = n * c["nodes"]
    kv = torch.randn(2, L, T, HK, D, device=DEV, generator=g).to(dt)
    st["k"], st["v"] = kv[0], kv[1]
    if own:
        from respect_b200.decoding.kv_pages import PagedKVCache
        st["cache"] = PagedKVCache.from_state(st["store"], st["table"], st["lengths"], st["held"], st["refs"])
    return st


def _prepare_logprobs(c, g):
    """Logits of a trained head: a broad bulk, a few strong candidates a row, and ties."""
    rows, V, dt = c["rows"], c["V"], DTYPES[c["dtype"]]
    x = torch.empty(rows, V, device=DEV, dtype=dt)
    for r in range(0, rows, 256):
        y = torch.randn(min(256, rows - r), V, device=DEV, generator=g) * 2.0
        hot = torch.randint(0, V, (y.shape[0], 8), device=DEV, generator=g)
        y.scatter_add_(1, hot, torch.rand(y.shape[0], 8, device=DEV, generator=g) * 14.0)
        x[r:r + 256] = y.to(dt)
    if c["size"] == 0:
        tokens = torch.randint(0, V, (rows,), device=DEV, generator=g)
    else:   # a given token is one that the choice may take
        tokens = torch.randint(0, V - c["size"], (rows,), device=DEV, generator=g)
        tokens = torch.where(tokens >= c["offset"], tokens + c["size"], tokens)
    best = x.float()[:, :c["offset"]].argmax(1) if c["offset"] > 0 else None
    if best is not None:                # half of the given tokens are likely ones
        tokens = torch.where(torch.arange(rows, device=DEV) % 2 == 0, best, tokens)
    return dict(logits=x, tokens=tokens)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    make = {"prompt": _prepare_prompt, "paged": _prepare_paged, "pages_fork": _prepare_pages,
            "pages_round": _prepare_pages, "logprobs": _prepare_logprobs}[op]
    return dict(make(case, g), case=case)


# ---------------------------------------------------------------- plain forms
def _plain_prompt(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    H, HK = c["H"], c["HK"]
    G = H // HK
    out = torch.empty(q.shape, device=DEV, dtype=q.dtype)
    at = 0
    for n in s["lens"]:
        for h in range(HK):
            kh, vh = k[at:at + n, h].float(), v[at:at + n, h].float()
            rows = 2048 if n <= 8192 else 512
            for r in range(0, n, rows):
                e = min(n, r + rows)
                qh = q[at + r:at + e, h * G:(h + 1) * G].float().transpose(0, 1)          # [G, rows, D]
                sc = torch.matmul(qh, kh[:e].T) * D ** -0.5
                future = torch.arange(e, device=DEV)[None, :] > torch.arange(r, e, device=DEV)[:, None]
                sc.masked_fill_(future, float("-inf"))
                sc -= sc.amax(-1, keepdim=True)
                sc.exp_()
                o = torch.matmul(sc, vh[:e]) / sc.sum(-1, keepdim=True)
                out[at + r:at + e, h * G:(h + 1) * G] = o.transpose(0, 1).to(q.dtype)
        at += n
    return out


def _plain_paged(s):
    c, q = s["case"], s["q"]
    H, HK, ps = c["H"], c["HK"], c["page"]
    out = torch.zeros(q.shape, device=DEV, dtype=q.dtype)
    for b, n in enumerate(s["lens"]):
        if n == 0:
            continue
        pages = s["table"][b, :(n + ps - 1) // ps].long()
        kb = s["k"][pages].transpose(1, 2).reshape(-1, HK, D)[:n].float()                  # [n, HK, D]
        vb = s["v"][pages].transpose(1, 2).reshape(-1, HK, D)[:n].float()
        qb = q[b].float().reshape(HK, H // HK, D)
        sc = torch.einsum("hgd,nhd->hgn", qb, kb) * D ** -0.5
        p = torch.exp(sc - sc.amax(-1, keepdim=True))
        o = torch.einsum("hgn,nhd->hgd", p, vb) / p.sum(-1, keepdim=True)
        out[b] = o.reshape(H, D).to(q.dtype)
    return out


def _plain_drop(s, seq, length):
    """Keep `length` tokens of a sequence and give its other pages back."""
    ps = s["store"].shape[4]
    keep, held = (length + ps - 1) // ps, int(s["held"][seq])
    if keep < held:
        s["refs"][s["table"][seq, keep:held].long()] -= 1
        s["table"][seq, keep:held] = -1
        s["held"][seq] = keep
    s["lengths"][seq] = length


def _plain_reserve(s, seqs, counts):
    """Room for `counts` tokens after each sequence's own: new pages by the lowest free number,
    in the sequences' order; a partly filled page that others share is copied first, except by
    the last of those who ask when nobody else holds it."""
    ps = s["store"].shape[4]
    free = iter((s["refs"] == 0).nonzero()[:, 0].tolist())
    refs = s["refs"].tolist()
    for seq, count in zip(seqs, counts):
        n, held = int(s["lengths"][seq]), int(s["held"][seq])
        if n % ps and count:
            page = int(s["table"][seq, n // ps])
            if refs[page] > 1:
                new = next(free)
                s["store"][:, :, new, :, :n % ps] = s["store"][:, :, page, :, :n % ps]
                s["table"][seq, n // ps] = new
                s["refs"][page] -= 1
                s["refs"][new] = 1
                refs[page] -= 1
        for i in range(held, (n + count + ps - 1) // ps):
            new = next(free)
            s["table"][seq, i] = new
            s["refs"][new] = 1
            s["held"][seq] = i + 1


def _plain_write(s, seqs, counts):
    ps = s["store"].shape[4]
    at = 0
    for seq, count in zip(seqs, counts):
        pos = int(s["lengths"][seq]) + torch.arange(count, device=DEV)
        page = s["table"][seq][pos // ps].long()
        for i, x in enumerate((s["k"], s["v"])):
            s["store"][:, i, page, :, pos % ps] = x[:, at:at + count].transpose(0, 1)
        at += count


def _state(s):
    return {n: s[n] for n in ("store", "table", "lengths", "held", "refs")}


def _plain_fork(s):
    src, dst = s["src"].tolist(), s["dst"].tolist()
    ps = s["store"].shape[4]
    for d in dst:
        _plain_drop(s, d, 0)
    for a, d in zip(src, dst):
        n = int(s["lengths"][a])
        pages = s["table"][a, :(n + ps - 1) // ps]
        s["table"][d, :pages.numel()] = pages
        s["refs"][pages.long()] += 1
        s["held"][d], s["lengths"][d] = pages.numel(), n
    ones = [1] * len(dst)
    _plain_reserve(s, dst, ones)
    _plain_write(s, dst, ones)
    s["lengths"][s["dst"].long()] += 1
    return _state(s)


def _plain_round(s):
    ps = s["store"].shape[4]
    seqs, counts = s["seqs"].tolist(), s["nodes"].tolist()
    for seq, n in zip(seqs, s["base"].tolist()):
        _plain_drop(s, seq, n)
    _plain_reserve(s, seqs, counts)
    _plain_write(s, seqs, counts)
    for i, (seq, m) in enumerate(zip(seqs, s["accept"].tolist())):
        n = int(s["lengths"][seq])
        a = n + s["paths"][i, :m].long()
        b = n + torch.arange(m, device=DEV)
        row = s["table"][seq].long()
        s["store"][:, :, row[b // ps], :, b % ps] = s["store"][:, :, row[a // ps], :, a % ps].clone()
        _plain_drop(s, seq, n + m)
    return _state(s)


def _plain_logprobs(s):
    c = s["case"]
    parts = []
    for r in range(0, c["rows"], 256):
        x = s["logits"][r:r + 256].float()
        if c["size"]:
            x = x.clone()
            x[:, c["offset"]:c["offset"] + c["size"]] = float("-inf")
        z = x - x.amax(1, keepdim=True)
        e = torch.exp(z)
        total = e.sum(1, keepdim=True)
        lp = z - torch.log(total)
        entropy = -(torch.where(e > 0, lp, 0.0) * e).sum(1) / total[:, 0]
        out = [torch.gather(lp, 1, s["tokens"][r:r + 256, None])[:, 0], entropy]
        if c["top"]:
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]]
            out += [torch.gather(lp, 1, order), order]
        parts.append(out)
    return [torch.cat(p) for p in zip(*parts)]


# ---------------------------------------------------------------- this package's calls
def _own_prompt(s):
    from respect_b200.kernels.attention import prompt_attention
    return prompt_attention(s["q"], s["k"], s["v"], s["cu"])


def _own_paged(s):
    from respect_b200.kernels.attention import paged_attention
    return paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"])


def _own_fork(s):
    cache = s["cache"]
    cache.free(s["dst"])
    cache.fork(s["src"], s["dst"])
    cache.reserve(s["dst"], s["ones"])
    cache.write(s["k"], s["v"], s["dst"])
    cache.commit(s["dst"], s["ones"])
    return _state(s)


def _own_round(s):
    cache = s["cache"]
    cache.truncate(s["seqs"], s["base"])
    cache.reserve(s["seqs"], s["nodes"])
    cache.write(s["k"], s["v"], s["seqs"], s["cu"])
    cache.compact(s["seqs"], s["paths"], s["accept"])
    return _state(s)


def _own_logprobs(s):
    from respect_b200.decoding.acceptance import token_logprobs
    c = s["case"]
    r = token_logprobs(s["logits"], s["tokens"], c["top"], c["offset"], c["size"])
    return [r.logprob, r.entropy] + ([r.top_logprobs, r.top_ids] if c["top"] else [])


def run(state):
    forms = (_own_prompt, _own_paged, _own_fork, _own_round, _own_logprobs) if own else \
        (_plain_prompt, _plain_paged, _plain_fork, _plain_round, _plain_logprobs)
    at = ("prompt", "paged", "pages_fork", "pages_round", "logprobs").index(state["case"]["op"])
    return forms[at](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, op = case, case["op"]
    es = 4 if c["dtype"] == "f32" else 2
    if op == "prompt":
        lens = _ints(c["lens"])
        return {"bytes": sum(lens) * (2 * c["H"] + 2 * c["HK"]) * D * es + 4 * (len(lens) + 1),
                "flops": 4 * D * c["H"] * sum(n * (n + 1) // 2 for n in lens)}
    if op == "paged":
        lens = _ints(c["lens"])
        pages = sum((n + c["page"] - 1) // c["page"] for n in lens)
        return {"bytes": sum(lens) * 2 * c["HK"] * D * es + 2 * len(lens) * c["H"] * D * es + 4 * (pages + len(lens)),
                "flops": 4 * D * c["H"] * sum(lens)}
    if op == "logprobs":
        return {"bytes": c["rows"] * ((c["V"] - c["size"]) * es + 8 + 8 + 12 * c["top"]),
                "flops": 6 * c["rows"] * (c["V"] - c["size"])}
    lens, ps = _ints(c["lens"]), c["page"]
    slot = 2 * c["L"] * c["HK"] * D * es            # one token's K and V in every layer
    if op == "pages_fork":
        new = len(lens) * c["each"]
        copied = sum(n % ps for n in lens) * c["each"]
        tables = sum((n + ps - 1) // ps for n in lens) * (1 + c["each"]) * 4
        return {"bytes": 2 * slot * (copied + new) + tables, "flops": 0}
    moved = sum(_ints(c["accept"]))
    return {"bytes": 2 * slot * (len(lens) * c["nodes"] + moved) + 8 * len(lens) * (c["nodes"] // ps + 1), "flops": 0}


# ---------------------------------------------------------------- 64-bit results
def _exact_pages(case, s):
    """The state after one pass, with the tables worked out on the host and every moved slot in a list."""
    ps, pool = case["page"], s["refs"].tolist()
    rows, lengths = [[x for x in r if x >= 0] for r in s["table"].tolist()], s["lengths"].tolist()
    store, moves, fresh = s["store"].double(), [], []       # moves (from, to) and fresh (token, to), by (page, slot)
    lowest = [p for p, n in enumerate(pool) if n == 0]

    def take():
        pool[lowest[0]] = 1
        return lowest.pop(0)

    if case["op"] == "pages_fork":
        for t, (a, d) in enumerate(zip(s["src"].tolist(), s["dst"].tolist())):
            n = lengths[a]
            rows[d] = list(rows[a])
            if n % ps:      # the prompt keeps its own last page, so each sample has a copy of it
                old, rows[d][-1] = rows[d][-1], take()
                moves += [((old, i), (rows[d][-1], i)) for i in range(n % ps)]
            else:
                rows[d].append(take())
            for p in rows[d][:n // ps]:
                pool[p] += 1
            fresh.append((t, (rows[d][-1], n % ps)))
            lengths[d] = n + 1
    else:
        nodes = case["nodes"]
        for i, m in enumerate(s["accept"].tolist()):
            n, path = lengths[i], s["paths"][i].tolist()
            while len(rows[i]) * ps < n + nodes:
                rows[i].append(take())
            at = [(rows[i][x // ps], x % ps) for x in range(n, n + nodes)]
            fresh += [(i * nodes + j, at[j]) for j in range(nodes)]
            fresh += [(i * nodes + path[j], at[j]) for j in range(m)]     # later ones stand
            lengths[i] = n + m
            while (len(rows[i]) - 1) * ps >= n + m:
                pool[rows[i].pop()] = 0
    for what, src in ((moves, None), (fresh, (s["k"], s["v"]))):
        last = {to: a for a, to in what}
        if last:
            page, slot = (torch.tensor(x, device=DEV) for x in zip(*last))
            for kv in (0, 1):
                if src is None:
                    a, b = (torch.tensor(x, device=DEV) for x in zip(*last.values()))
                    val = s["store"][:, kv, a, :, b]
                else:
                    val = src[kv][:, torch.tensor(list(last.values()), device=DEV)].transpose(0, 1)
                store[:, kv, page, :, slot] = val.double()
    wide = s["table"].shape[1]
    return {"store": store, "table": _i32([r + [-1] * (wide - len(r)) for r in rows]), "lengths": _i32(lengths),
            "held": _i32([len(r) for r in rows]), "refs": _i32(pool)}


def exact(case, seed):
    """What run returns, from the definitions in 64 bits: a softmax written with its explicit weights."""
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["op"].startswith("pages"):
        return _exact_pages(case, s)
    if case["op"] == "logprobs":
        lo, hi, top = case["offset"], case["offset"] + case["size"], case["top"]
        rows = [[], [], [], []]
        for r in range(case["rows"]):
            x = s["logits"][r].double()
            keep = torch.cat((x[:lo], x[hi:]))
            lse = torch.logsumexp(keep, 0)
            p = torch.softmax(keep, 0)
            rows[0].append(x[s["tokens"][r]] - lse)
            rows[1].append(lse - (p * keep).sum())
            if top:
                best = torch.sort(keep, descending=True, stable=True)
                vals, ids = best.values[:top] - lse, best.indices[:top]
                rows[2].append(vals)
                rows[3].append(torch.where(ids >= lo, ids + (hi - lo), ids))
        if top and rows[2][0].numel() < top:
            return None
        return [torch.stack(x) for x in rows[:4 if top else 2]]
    lens, H, HK = s["lens"], case["H"], case["HK"]
    group = torch.arange(H, device=DEV) // (H // HK)
    out = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64)
    if case["op"] == "paged":
        ps = case["page"]
        for b, n in enumerate(lens):
            t = torch.arange(n, device=DEV)
            page, slot = s["table"][b].long()[t // ps], t % ps
            for h in range(H if n else 0):
                w = torch.softmax(s["k"][page, group[h], slot].double() @ s["q"][b, h].double() / math.sqrt(D), 0)
                out[b, h] = w @ s["v"][page, group[h], slot].double()
        return out
    start = 0
    for n in lens:
        for h in range(H):
            qh = s["q"][start:start + n, h].double() / math.sqrt(D)
            kh, vh = (s[x][start:start + n, group[h]].double() for x in ("k", "v"))
            for a in range(0, n, 4096):
                b = min(n, a + 4096)
                w = qh[a:b] @ kh[:b].T
                w = w.masked_fill(~torch.ones(b - a, b, device=DEV, dtype=torch.bool).tril(a), -math.inf)
                out[start + a:start + b, h] = torch.softmax(w, 1) @ vh[:b]
        start += n
    return out
