"""Cases for the serving operators: appending to a paged KV cache with the
rotation applied, attention over it (sliding window, first tokens that stay
visible), attention of a batch that shares a long prefix, and token sampling.

``listed()`` names the measured cases and ``draw(rng)`` gives more of the same
ranges; ``prepare(case, seed)`` makes the inputs on the GPU, ``run(state)`` is
one pass (the plain form in torch operations, or with ``own`` the framework's
operators), ``exact(case, seed)`` the definition in 64 bits, and ``work(case)``
the bytes and operations a pass cannot do without.
"""
import math
import random

import torch

own = False

D = 128            # head dimension of every configuration
VOCAB = 151936     # vocabulary of the benchmarked configurations
THETA = 1e6        # rotary base of the 0.6B and 8B configurations
EPS = 1e-6
BF16 = torch.bfloat16


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # one token of one sequence: what a step of a chat adds to the cache
        _append("append one token", 32, 8, page=16, seqs=1, q=(1, 1), kv=(4097, 4097)),
        # a decode step of a busy server: one token for each of many ragged sequences
        _append("append a decode batch", 32, 8, page=16, seqs=96, q=(1, 1), kv=(1, 2000)),
        # prompts that are prefilled together, packed, in a buffer with unused rows at its end
        _append("append packed prompts", 32, 8, page=64, seqs=5, q=(900, 2300), kv=(900, 4000), pad=37),
        # the smallest model's decode step at a short context: only latency counts
        _attend("attend short decode", 16, 8, page=16, seqs=1, q=(1, 1), kv=(512, 512)),
        # a decode step of a busy server over full attention: streams the whole cache
        _attend("attend decode batch", 32, 8, page=64, seqs=64, q=(1, 1), kv=(130, 16384)),
        # a windowed layer far into long documents, with the first tokens kept
        _attend("attend windowed decode", 32, 8, page=16, seqs=32, q=(1, 1), kv=(9000, 131072),
                window=4096, sinks=4),
        # a long prompt's next chunk, running beside decoding sequences (mixed batch), windowed
        _attend("attend windowed chunk", 32, 8, page=32, seqs=9, q=(1, 1), kv=(70, 5000), chunk=1999, chunk_kv=9001,
                window=2048, sinks=64),
        # a whole long prompt
        _attend("attend prompt", 32, 8, page=64, seqs=1, q=(8100, 8100), kv=(8100, 8100)),
        # a handful of samples of one short question, 4 heads (one rank of several)
        _prefix("prefix few", 4, 1, page=16, seqs=6, prefix=1000, q=(1, 1), kv=(1, 90)),
        # a server whose requests all start with the same long document
        _prefix("prefix many", 32, 8, page=64, seqs=64, prefix=32768, q=(1, 1), kv=(1, 700)),
        # one sequence's next token, with the usual chat settings
        _sample("sample one", 1, "bf16", temperature=(0.7, 0.7), top_k=(20, 20), top_p=(0.8, 0.8)),
        # a decode batch whose requests each bring their own settings
        _sample("sample batch", 192, "fp32", temperature=(0.3, 1.5), top_k=(0, 2000), top_p=(0.5, 1.0),
                min_p=(0.0, 0.1), banned=0.01),
    ]


def _append(name, hq, hkv, page, seqs, q, kv, pad=0, layout=1):
    return {"name": name, "op": "append", "hq": hq, "hkv": hkv, "page": page, "seqs": seqs, "q_lo": q[0], "q_hi": q[1],
            "kv_lo": kv[0], "kv_hi": kv[1], "chunk": 0, "chunk_kv": 0, "prefix": 0, "pad": pad, "layout": layout}


def _attend(name, hq, hkv, page, seqs, q, kv, chunk=0, chunk_kv=0, window=0, sinks=0, pad=0, layout=2):
    return {"name": name, "op": "attend", "hq": hq, "hkv": hkv, "page": page, "seqs": seqs, "q_lo": q[0], "q_hi": q[1],
            "kv_lo": kv[0], "kv_hi": kv[1], "chunk": chunk, "chunk_kv": chunk_kv, "prefix": 0, "window": window,
            "sinks": sinks, "pad": pad, "layout": layout}


def _prefix(name, hq, hkv, page, seqs, prefix, q, kv, pad=0, layout=3):
    return {"name": name, "op": "prefix", "hq": hq, "hkv": hkv, "page": page, "seqs": seqs, "q_lo": q[0], "q_hi": q[1],
            "kv_lo": kv[0], "kv_hi": kv[1], "chunk": 0, "chunk_kv": 0, "prefix": prefix, "pad": pad, "layout": layout}


def _sample(name, rows, dtype, temperature, top_k=(0, 0), top_p=(1.0, 1.0), min_p=(0.0, 0.0), banned=0.0, vocab=VOCAB):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "t_lo": temperature[0],
            "t_hi": temperature[1], "k_lo": top_k[0], "k_hi": top_k[1], "p_lo": top_p[0], "p_hi": top_p[1],
            "m_lo": min_p[0], "m_hi": min_p[1], "banned": banned}


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "prefix", "sample"])
    hq, hkv = rng.choice([(32, 8), (16, 8), (8, 4), (4, 1), (32, 8)])
    page = rng.choice([16, 32, 64, 128])
    layout = rng.randrange(1 << 30)
    pad = rng.choice([0, 0, rng.randrange(1, 40)])
    if op == "append":
        tokens = _log_int(rng, 1, 8000)
        seqs = _log_int(rng, 1, min(tokens, 128))
        q_hi = max(1, tokens // seqs)
        q_lo = rng.choice([q_hi, max(1, q_hi // 3), 0 if seqs > 1 else q_hi])
        c = _append("", hq, hkv, page, seqs, (q_lo, q_hi), (max(1, q_hi), q_hi + rng.randrange(1, 2500)), pad, layout)
    elif op == "attend":
        window, sinks = rng.choice([(0, 0), (0, 0), (_log_int(rng, 1, 8192), rng.choice([0, 1, 4, 64, 130]))])
        kind = rng.choice(["decode", "verify", "chunk", "mixed"])
        if kind in ("decode", "verify"):
            n = 1 if kind == "decode" else rng.randrange(2, 17)
            kv_hi = _log_int(rng, 16, 131072)
            seqs = _log_int(rng, 1, max(1, min(128, 524288 // kv_hi)))
            c = _attend("", hq, hkv, page, seqs, (n, n), (min(kv_hi, max(n, kv_hi // 8)), max(n, kv_hi)),
                        window=window, sinks=sinks, pad=pad, layout=layout)
        elif kind == "chunk":
            tokens = _log_int(rng, 17, 8000)
            seqs = rng.randrange(1, 5)
            n = max(1, tokens // seqs)
            c = _attend("", hq, hkv, page, seqs, (max(1, n // 2), n), (n, n + rng.choice([0, rng.randrange(4000)])),
                        window=window, sinks=sinks, pad=pad, layout=layout)
        else:
            chunk = _log_int(rng, 16, 2500)
            c = _attend("", hq, hkv, page, _log_int(rng, 2, 40), (0, 1), (1, _log_int(rng, 20, 10000)),
                        chunk=chunk, chunk_kv=chunk + rng.randrange(8000), window=window, sinks=sinks, pad=pad,
                        layout=layout)
    elif op == "prefix":
        seqs = _log_int(rng, 1, 128)
        n = rng.choice([1, 1, 1, rng.randrange(2, 9)])
        c = _prefix("", hq, hkv, page, seqs, _log_int(rng, 1, 32768), (n, n),
                    (n, n + _log_int(rng, 1, 1000)), pad, layout)
    else:
        rows = _log_int(rng, 1, 192)
        c = _sample("", rows, rng.choice(["bf16", "fp32"]), (0.0 if rng.random() < 0.2 else 0.3, rng.uniform(0.5, 2.0)),
                    rng.choice([(0, 0), (1, 64), (0, 5000)]), rng.choice([(1.0, 1.0), (0.3, 1.0), (0.9, 0.95)]),
                    rng.choice([(0.0, 0.0), (0.0, 0.2)]), rng.choice([0.0, 0.02]),
                    rng.choice([VOCAB, 4096, _log_int(rng, 100, VOCAB)]))
    del c["name"]
    return c


def _lengths(case):
    """(queries, cached tokens) of each sequence; a case's own numbers fix them."""
    rng = random.Random(case["layout"])
    out = []
    for i in range(case["seqs"]):
        n = rng.randint(case["q_lo"] if i else max(1, case["q_lo"]), case["q_hi"])
        kv = case["kv_lo"] + int((case["kv_hi"] - case["kv_lo"]) * rng.random() ** 2 + 0.5)
        if i == 0 and case["kv_hi"] > case["kv_lo"]:
            kv = case["kv_hi"]
        out.append((n, max(n, kv)))
    if case["chunk"]:
        out.insert(len(out) // 2, (case["chunk"], max(case["chunk"], case["chunk_kv"])))
    return out


def _seen(case, n, kv):
    """(keys some query of the sequence sees, sum over its queries of the keys seen)."""
    w, s = case.get("window", 0), case.get("sinks", 0)
    first = kv - n
    if w == 0:
        return kv, n * first + n * (n + 1) // 2
    lo = max(0, first - w + 1)
    union = kv - lo + min(s, lo) if n else 0
    total = 0
    for i in range(n):
        p = first + i
        a = max(0, p - w + 1)
        total += p + 1 - a + min(s, a)
    return union, total


def work(case):
    if case["op"] == "sample":
        size = 2 if case["dtype"] == "bf16" else 4
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * 28, "flops": 4 * n}
    hq, hkv = case["hq"], case["hkv"]
    lens = _lengths(case)
    tokens = sum(n for n, _ in lens)
    if case["op"] == "append":
        per = (2 * hq + 4 * hkv) * D * 2 + 2 * D * 2
        return {"bytes": tokens * per, "flops": tokens * (hq + hkv) * D * 8}
    kv_bytes, pairs = 0, 0
    for n, kv in lens:
        union, total = _seen(case, n, kv)
        kv_bytes += (union if n else 0) * hkv * D * 4
        pairs += total
    kv_bytes += case["prefix"] * hkv * D * 4
    pairs += case["prefix"] * tokens
    return {"bytes": kv_bytes + 2 * tokens * hq * D * 2, "flops": 4 * D * hq * pairs}


# ------------------------------------------------------------------ the inputs
def _tables(positions, device):
    """cos and sin rows of positions 0..positions-1 in bf16, angles in 64 bits."""
    inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=device) / D)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv[None]
    angle = torch.cat((angle, angle), dim=1)
    return angle.cos().to(BF16), angle.sin().to(BF16)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=BF16):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * scale).to(dtype)

    st = dict(case=case)
    if case["op"] == "sample":
        r, v = case["rows"], case["vocab"]
        # a language model's logits: a broad body, and for each row a few likely tokens
        x = torch.randn(r, v, generator=gen, device=dev) * 2.2
        likely = torch.randint(0, v, (r, 24), generator=gen, device=dev)
        x.scatter_add_(1, likely, 9 * torch.rand(r, 24, generator=gen, device=dev))
        if case["banned"]:
            x.masked_fill_(torch.rand(r, v, generator=gen, device=dev) < case["banned"], float("-inf"))
        st["logits"] = x.to(BF16) if case["dtype"] == "bf16" else x
        st["uniforms"] = torch.rand(r, generator=gen, device=dev)

        def spread(lo, hi):
            return lo + (hi - lo) * torch.rand(r, generator=gen, device=dev)

        st["temperature"] = spread(case["t_lo"], case["t_hi"])
        if case["t_lo"] == 0.0:  # some rows are greedy
            st["temperature"] = torch.where(st["temperature"] < 0.3, torch.zeros_like(st["temperature"]),
                                            st["temperature"])
        st["top_k"] = torch.randint(case["k_lo"], case["k_hi"] + 1, (r,), generator=gen, device=dev, dtype=torch.int32)
        st["top_p"] = spread(case["p_lo"], case["p_hi"])
        st["min_p"] = spread(case["m_lo"], case["m_hi"])
        return st

    hq, hkv, page, prefix = case["hq"], case["hkv"], case["page"], case["prefix"]
    lens = _lengths(case)
    tokens = sum(n for n, _ in lens)
    rows = tokens + case["pad"]
    own_pages = [-(-kv // page) for _, kv in lens]
    prefix_pages = -(-prefix // page)
    pages = sum(own_pages) + prefix_pages + 3
    ids = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    width = max(own_pages) + 1
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(own_pages):
        table[b, :n] = ids[at:at + n]
        at += n
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    st.update(lens=lens, starts=starts, page_table=table,
              q_start=torch.tensor(starts, dtype=torch.int32, device=dev),
              kv_lens=torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=dev),
              k_pages=normal(pages, hkv, page, D), v_pages=normal(pages, hkv, page, D),
              out=torch.zeros(rows, hq, D, dtype=BF16, device=dev))
    if case["op"] == "append":
        st["qkv"] = normal(rows, (hq + 2 * hkv) * D, scale=1.5)
        st["q_norm"] = (1 + 0.2 * torch.randn(D, generator=gen, device=dev)).to(BF16)
        st["k_norm"] = (1 + 0.2 * torch.randn(D, generator=gen, device=dev)).to(BF16)
        st["cos"], st["sin"] = _tables(max(kv for _, kv in lens), dev)
    else:
        st["q"] = normal(rows, hq, D, scale=1.4)
        st["max_queries"] = max(n for n, _ in lens)
    if case["op"] == "prefix":
        st["prefix_table"] = ids[at:at + prefix_pages].contiguous()
    return st


# ------------------------------------------------------------------- one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    from hackthenorth_b200 import ops

    case = st["case"]
    if case["op"] == "append":
        q = ops.rope_paged_append(st["qkv"], st["q_norm"], st["k_norm"], st["cos"], st["sin"], st["k_pages"],
                                  st["v_pages"], st["page_table"], st["q_start"], st["kv_lens"], eps=EPS, out=st["out"])
        return q, st["k_pages"], st["v_pages"]
    if case["op"] == "attend":
        return ops.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["page_table"], st["q_start"],
                                   st["kv_lens"], window=case["window"], sinks=case["sinks"],
                                   max_queries=st["max_queries"], out=st["out"])
    if case["op"] == "prefix":
        return ops.shared_prefix_attention(st["q"], st["k_pages"], st["v_pages"], st["prefix_table"], case["prefix"],
                                           st["page_table"], st["q_start"], st["kv_lens"],
                                           max_queries=st["max_queries"], out=st["out"])
    return ops.sample_token(st["logits"], st["uniforms"], temperature=st["temperature"], top_k=st["top_k"],
                            top_p=st["top_p"], min_p=st["min_p"])


def _run_plain(st):
    op = st["case"]["op"]
    if op == "append":
        return _plain_append(st)
    if op == "sample":
        return _plain_sample(st)
    return _plain_attend(st)


def _plain_append(st):
    case = st["case"]
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    rows = st["starts"][-1]
    t = torch.arange(rows, device="cuda")
    b = torch.searchsorted(st["q_start"].long(), t, right=True) - 1
    pos = st["kv_lens"].long()[b] - st["q_start"].long()[b + 1] + t
    cos, sin = st["cos"][pos].float()[:, None], st["sin"][pos].float()[:, None]
    x = st["qkv"][:rows].float().view(rows, hq + 2 * hkv, D)

    def turn(y, gain):
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * gain.float()
        half = torch.cat((-y[..., D // 2:], y[..., :D // 2]), dim=-1)
        return (y * cos + half * sin).to(BF16)

    st["out"][:rows] = turn(x[:, :hq], st["q_norm"])
    page_ids = st["page_table"][b, pos // page].long()
    st["k_pages"][page_ids, :, pos % page] = turn(x[:, hq:hq + hkv], st["k_norm"])
    st["v_pages"][page_ids, :, pos % page] = x[:, hq + hkv:].to(BF16)
    return st["out"], st["k_pages"], st["v_pages"]


def _gather(pages, ids, count, heads):
    """Keys or values 0..count-1 of some heads, in 32 bits: [heads, count, D]."""
    return pages[ids.long(), heads].transpose(0, 1).reshape(heads.stop - heads.start, -1, D)[:, :count].float()


def _plain_attend(st):
    case = st["case"]
    hq, hkv, page, prefix = case["hq"], case["hkv"], case["page"], case["prefix"]
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    G = hq // hkv
    for b, (n, kv) in enumerate(st["lens"]):
        if n == 0:
            continue
        a = st["starts"][b]
        lo = max(0, kv - n - window + 1) // page * page if window else 0
        own_ids = st["page_table"][b, :-(-kv // page)]
        keep = torch.arange(kv, device="cuda")
        if lo > sinks:  # leave out what no query of the sequence sees
            head_pages = -(-sinks // page)
            own_ids = torch.cat((own_ids[:head_pages], own_ids[lo // page:]))
            keep = torch.cat((keep[:head_pages * page], keep[lo:]))
        pos = torch.arange(kv - n, kv, device="cuda")[:, None]
        seen = keep[None] <= pos
        if window:
            seen &= (keep[None] > pos - window) | (keep[None] < sinks)
        if prefix:
            seen = torch.cat((torch.ones(n, prefix, dtype=torch.bool, device="cuda"), seen), dim=1)
        step = max(1, min(hkv, 2 ** 28 // (n * G * seen.shape[1])))  # heads at a time: scores of 1 GB
        for g in range(0, hkv, step):
            heads = slice(g, min(hkv, g + step))
            k = _gather(st["k_pages"], own_ids, keep.numel(), heads)
            v = _gather(st["v_pages"], own_ids, keep.numel(), heads)
            if prefix:
                k = torch.cat((_gather(st["k_pages"], st["prefix_table"], prefix, heads), k), dim=1)
                v = torch.cat((_gather(st["v_pages"], st["prefix_table"], prefix, heads), v), dim=1)
            q = st["q"][a:a + n].float().view(n, hkv, G, D)[:, heads].transpose(0, 1)
            s = (q.reshape(-1, n * G, D) @ k.transpose(1, 2)).view(-1, n, G, seen.shape[1]) * D ** -0.5
            s = s.masked_fill(~seen[:, None], float("-inf"))
            s = torch.exp(s - s.amax(-1, keepdim=True))
            y = s.view(-1, n * G, seen.shape[1]) @ v / s.sum(-1).view(-1, n * G, 1)
            st["out"][a:a + n].view(n, hkv, G, D)[:, heads] = y.view(-1, n, G, D).transpose(0, 1).to(BF16)
    return st["out"]


def _plain_sample(st):
    """Ranks by falling logit (ties: lowest index first); the first top_k of
    them; of those the ones before which less than top_p of their mass lies;
    of those the ones with at least min_p of the largest weight. The token is
    the first, by index, at which the running mass passes uniform * mass."""
    x = st["logits"].double()
    t = st["temperature"].double()[:, None]
    top = x.amax(1, keepdim=True)
    w = torch.exp((x - top) / torch.where(t > 0, t, torch.ones_like(t)))
    w, order = torch.sort(w, dim=1, descending=True, stable=True)
    # equal weights of unequal logits (both 0) have no mass, so their order does not matter
    rank = torch.arange(x.shape[1], device="cuda")[None]
    k = st["top_k"].long()[:, None]
    k = torch.where(k > 0, k, torch.full_like(k, x.shape[1]))
    w = w * (rank < k)
    before = w.cumsum(1) - w
    p = st["top_p"].double()[:, None]
    w = w * ((before < p * w.sum(1, keepdim=True)) | (p >= 1) | (rank == 0))
    w = w * (w >= st["min_p"].double()[:, None])
    w = torch.zeros_like(w).scatter_(1, order, w)
    cum = w.cumsum(1)
    target = st["uniforms"].double()[:, None] * cum[:, -1:]
    token = (cum > target).int().argmax(1)
    return torch.where(t[:, 0] > 0, token, x.argmax(1))


# ----------------------------------------------------------- in 64 bits, apart
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    if case["op"] == "append":
        return _exact_append(st)
    return _exact_attend(st)


def _slots(st, b, positions):
    """Rows of the pool, flattened to [page * head * slot], of one sequence's positions and head 0."""
    case = st["case"]
    ids = st["page_table"][b].long()[torch.div(positions, case["page"], rounding_mode="floor")]
    return ids * case["hkv"] * case["page"] + positions.remainder(case["page"])


def _exact_append(st):
    case = st["case"]
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    keys, values = st["k_pages"].double().view(-1, D), st["v_pages"].double().view(-1, D)
    seq = torch.repeat_interleave(torch.arange(len(st["lens"])), torch.tensor([n for n, _ in st["lens"]]))
    for b in sorted(set(seq.tolist())):
        n, kv = st["lens"][b]
        first = st["starts"][b]
        p = torch.arange(n, device="cuda") + (kv - n)
        cos, sin = st["cos"].double()[p, :D // 2], st["sin"].double()[p, :D // 2]
        heads = st["qkv"][first:first + n].double().split(D, dim=1)
        where = _slots(st, b, p)
        for h, x in enumerate(heads):
            if h < hq + hkv:
                gain = (st["q_norm"] if h < hq else st["k_norm"]).double()
                x = gain * x / torch.sqrt(x.square().sum(1, keepdim=True) / D + EPS)
                u, v = x[:, :D // 2], x[:, D // 2:]
                x = torch.cat((u * cos - v * sin, v * cos + u * sin), dim=1)
            if h < hq:
                out[first:first + n, h] = x
            elif h < hq + hkv:
                keys[where + (h - hq) * page] = x
            else:
                values[where + (h - hq - hkv) * page] = x
    return out, keys.view(st["k_pages"].shape), values.view(st["v_pages"].shape)


def _exact_attend(st):
    """One query block at a time: the softmax's weights over the visible keys."""
    case = st["case"]
    hq, hkv, page, prefix = case["hq"], case["hkv"], case["page"], case["prefix"]
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    pairs = sum(n * kv for n, kv in st["lens"]) + prefix * st["starts"][-1]
    if pairs * hq > 6e9:  # would take too long in 64 bits
        return None
    G = hq // hkv
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    flat_k, flat_v = st["k_pages"].view(-1, D), st["v_pages"].view(-1, D)
    for b, (n, kv) in enumerate(st["lens"]):
        for i0 in range(0, n, 1024):
            i1 = min(n, i0 + 1024)
            p = torch.arange(i0, i1, device="cuda") + (kv - n)
            c = torch.arange(int(p[-1]) + 1, device="cuda")
            if window:
                c = c[(c > kv - n + i0 - window) | (c < sinks)]
            mask = c[None] > p[:, None]
            if window:
                mask |= (p[:, None] - c[None] >= window) & (c[None] >= sinks)
            where = _slots(st, b, c)
            if prefix:
                z = torch.arange(prefix, device="cuda")
                shared = st["prefix_table"].long()[z // page] * hkv * page + z % page
                where = torch.cat((shared, where))
                mask = torch.nn.functional.pad(mask, (prefix, 0))
            for h in range(hkv):
                k, v = flat_k[where + h * page].double(), flat_v[where + h * page].double()
                for j in range(h * G, (h + 1) * G):
                    a = st["q"][st["starts"][b] + i0:st["starts"][b] + i1, j].double() @ k.T / math.sqrt(D)
                    a[mask] = -math.inf
                    out[st["starts"][b] + i0:st["starts"][b] + i1, j] = torch.softmax(a, dim=1) @ v
    return out


def _exact_sample(st):
    """Row by row: the kept set grows from the most likely token downwards."""
    case = st["case"]
    if case["rows"] * case["vocab"] > 4e7:
        return None
    tokens = []
    for r in range(case["rows"]):
        x = st["logits"][r].double()
        t = float(st["temperature"][r].double())
        if not t > 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            continue
        idx = torch.argsort(-x, stable=True)
        k = int(st["top_k"][r])
        idx = idx[:k] if k > 0 else idx
        weight = torch.exp((x[idx] - x[idx[0]]) / t)
        p = float(st["top_p"][r].double())
        if p < 1:
            total = float(weight.sum())
            ahead = torch.cat((weight.new_zeros(1), weight.cumsum(0)[:-1]))
            count = max(1, int((ahead < p * total).sum()))
            idx, weight = idx[:count], weight[:count]
        keep = weight >= float(st["min_p"][r].double())
        idx, weight = idx[keep], weight[keep]
        idx, by_index = idx.sort()
        run_mass = weight[by_index].cumsum(0)
        hit = int(torch.searchsorted(run_mass, float(st["uniforms"][r].double()) * run_mass[-1], right=True))
        tokens.append(int(idx[min(hit, idx.numel() - 1)]))
    return torch.tensor(tokens, dtype=torch.int64, device="cuda")
