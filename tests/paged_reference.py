"""Plain 64-bit forms of the paged-cache operators and their tests' inputs."""
import torch

BF16 = torch.bfloat16
D = 128


def make_batch(lens, hq, hkv, page, seed, device, pad=0, spare=2, scale=1.0, prefix=0):
    """A paged batch of sequences with (queries, cached keys) ``lens``: pools,
    tables and q, all from the seed; pages in random order. ``pages`` keeps the
    table that ``table`` starts as (a test may spoil entries that no key needs)."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-kv // page) for _, kv in lens]
    n_prefix = -(-prefix // page)
    pages = sum(counts) + n_prefix + spare
    ids = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = ids[at:at + c]
        at += c
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    rows = starts[-1] + pad
    gd = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gd, device=device).to(BF16)
    return dict(lens=lens, hq=hq, hkv=hkv, page=page, starts=starts, rows=rows, prefix=prefix,
                prefix_table=ids[at:at + n_prefix].to(device), spare=ids[at + n_prefix:].tolist(),
                q=(scale * torch.randn(rows, hq, D, generator=gd, device=device)).to(BF16),
                k=rnd(pages, hkv, page, D), v=rnd(pages, hkv, page, D), table=table.to(device), pages=table.clone().to(device),
                q_start=torch.tensor(starts, dtype=torch.int32, device=device),
                kv_lens=torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=device))


def keys_of(pool, ids, count, head):
    ids = ids[:-(-count // pool.shape[2])]
    return pool[ids.long(), head].reshape(-1, D)[:count].double()


def attention64(bt, window=0, sinks=0):
    """(result, sum of weight * |value|) in 64 bits; rows of no sequence are NaN."""
    hq, hkv, page, prefix = bt["hq"], bt["hkv"], bt["page"], bt["prefix"]
    G = hq // hkv
    out = torch.full((bt["rows"], hq, D), float("nan"), dtype=torch.float64, device=bt["q"].device)
    mag = out.clone()
    for b, (n, kv) in enumerate(bt["lens"]):
        if n == 0:
            continue
        a = bt["starts"][b]
        if kv + prefix == 0:
            out[a:a + n] = mag[a:a + n] = 0.0
            continue
        p = torch.arange(kv - n, kv, device=out.device)[:, None]
        c = torch.arange(kv, device=out.device)[None]
        seen = c <= p
        if window:
            seen = seen & ((c > p - window) | (c < sinks))
        seen = torch.cat((torch.ones(n, prefix, dtype=torch.bool, device=out.device), seen), 1)
        for g in range(hkv):
            k = torch.cat((keys_of(bt["k"], bt["prefix_table"], prefix, g), keys_of(bt["k"], bt["pages"][b], kv, g)))
            v = torch.cat((keys_of(bt["v"], bt["prefix_table"], prefix, g), keys_of(bt["v"], bt["pages"][b], kv, g)))
            dead = ~seen.any(0)
            k, v = k.masked_fill(dead[:, None], 0.0), v.masked_fill(dead[:, None], 0.0)
            s = torch.einsum("ngd,kd->ngk", bt["q"][a:a + n, g * G:(g + 1) * G].double(), k) / D ** 0.5
            s = s.masked_fill(~seen[:, None], float("-inf"))
            w = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
            w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
            out[a:a + n, g * G:(g + 1) * G] = w @ v
            mag[a:a + n, g * G:(g + 1) * G] = w @ v.abs()
    return out, mag


def attention_bound(ref, mag):
    """Half a bf16 step of the result (2^-8), P's rounding to bf16 (2^-8 of the
    summed magnitudes), and what fp32 leaves: a score is a sum of 128 products
    of at most a few units, off by less than 128 * 2^-24 * 2^5 = 2^-12, and so
    is, relatively, its weight; the joins and sums are far below that."""
    return 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -11) * mag + 1e-30
