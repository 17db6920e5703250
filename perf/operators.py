"""What is measured of the block-sparse and paged attention operators: cases, inputs, plain forms and exact values.

Four operators:

  append   new keys and values go into a paged cache, keys (and the queries beside them) rotated by their positions, the
           pages' key sums brought up to date
  select   the blocks of keys that every query block reads: the largest products of the summed queries with the blocks'
           mean keys
  train    attention of every query block over its listed blocks, with the gradients of q, k and v
  attend   attention of the newest tokens of every sequence over a paged cache, over all pages or the listed ones

`run` computes them in plain torch operations; with `own` set it calls cuspamm_b200.
"""
import math

import torch

own = False

BF16, FP16 = "bf16", "fp16"
DTYPES = {BF16: torch.bfloat16, FP16: torch.float16}


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one decoding step of a busy server: 64 sequences grow by a token each
        dict(name="append_step", op="append", dtype=BF16, batch=64, new=1, length=2048, heads=32, kv_heads=8, dim=128,
             block=64, rotary=128, interleaved=False, ragged=True),
        # prompts of several requests written at once, half of each head rotated, neighbouring pairs
        dict(name="append_prompts", op="append", dtype=FP16, batch=5, new=4001, length=4001, heads=32, kv_heads=4,
             dim=128, block=32, rotary=64, interleaved=True, ragged=True),
        # lists of a training batch of three documents, one list for every 64 queries
        dict(name="select_train", op="select", paged=False, dtype=BF16, batch=3, new=16384, length=16384, heads=32,
             kv_heads=8, dim=128, block=64, query_block=64, n_select=16, n_first=1, n_local=2, ragged=True, causal=True),
        # a list for every single query of a long document
        dict(name="select_each_query", op="select", paged=False, dtype=FP16, batch=1, new=8192, length=8192, heads=64,
             kv_heads=4, dim=128, block=64, query_block=1, n_select=16, n_first=1, n_local=2, ragged=False, causal=True),
        # one decoding step over long contexts: every sequence's newest token picks its pages
        dict(name="select_step", op="select", paged=True, dtype=BF16, batch=16, new=1, length=65537, heads=32,
             kv_heads=8, dim=128, block=64, query_block=1, n_select=32, n_first=1, n_local=2, ragged=True, causal=True),
        # training step of a long batch, q, k and v cut from one fused projection
        dict(name="train_blocks", op="train", dtype=BF16, batch=3, new=8192, length=8192, heads=32, kv_heads=8, dim=128,
             block=64, query_block=64, n_select=16, ragged=True, causal=True, fused=True),
        # training step where every query has a list of its own, sixteen query heads to a key head
        dict(name="train_each_query", op="train", dtype=FP16, batch=2, new=2999, length=2999, heads=32, kv_heads=2,
             dim=128, block=64, query_block=1, n_select=16, ragged=True, causal=True, fused=False),
        # a small encoder: heads of 64, no mask, no shared heads, an odd length
        dict(name="train_encoder", op="train", dtype=BF16, batch=4, new=1021, length=1021, heads=12, kv_heads=12, dim=64,
             block=32, query_block=128, n_select=12, ragged=True, causal=False, fused=True),
        # the least there is: one sequence, one token, a page and a token of context
        dict(name="attend_first", op="attend", dtype=BF16, batch=1, new=1, length=65, heads=8, kv_heads=2, dim=64,
             block=64, query_block=1, n_select=0, ragged=False),
        # decoding step of 32 sequences over everything that they hold
        dict(name="attend_step", op="attend", dtype=BF16, batch=32, new=1, length=16384, heads=32, kv_heads=8, dim=128,
             block=64, query_block=1, n_select=0, ragged=True),
        # decoding step over the pages that were selected
        dict(name="attend_step_listed", op="attend", dtype=FP16, batch=16, new=1, length=32769, heads=64, kv_heads=4,
             dim=128, block=64, query_block=1, n_select=32, ragged=True),
        # chunks of two long prompts over what the cache holds of them already
        dict(name="attend_chunk", op="attend", dtype=BF16, batch=2, new=1024, length=32768, heads=32, kv_heads=8, dim=128,
             block=64, query_block=64, n_select=0, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "select", "train", "attend"])
    c = dict(op=op, dtype=rng.choice([BF16, FP16]), dim=rng.choice([64, 128]), block=rng.choice([16, 32, 64, 128]),
             ragged=rng.random() < 0.75)
    c["kv_heads"] = rng.choice([1, 2, 4, 8])
    c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 8, 16] if c["kv_heads"] < 8 else [1, 2, 4])
    if op == "append":
        c["batch"] = _log(rng, 1, 64)
        c["new"] = _log(rng, 1, max(2, 16000 // c["batch"]))
        c["length"] = c["new"] + (0 if rng.random() < 0.3 else _log(rng, 1, 2048))
        c["rotary"] = rng.choice([0, c["dim"] // 2, c["dim"]])
        c["interleaved"] = rng.random() < 0.5
    elif op == "select":
        c["paged"] = rng.random() < 0.5
        c["batch"] = _log(rng, 1, 16 if c["paged"] else 4)
        c["query_block"] = rng.choice([1, 16, 64, 128])
        c["n_first"], c["n_local"] = rng.choice([0, 1, 2]), rng.choice([1, 2])
        must = c["n_first"] + c["n_local"] + (c["query_block"] + c["block"] - 2) // c["block"]
        c["n_select"] = must + _log(rng, 1, 16)
        least = c["block"] * (2 * c["n_select"] + 8)        # so long that there is something to choose
        c["length"] = _log(rng, least, max(2 * least, 65000 if c["paged"] else 8192))
        c["new"] = c["length"]
        if c["paged"]:
            c["new"] = 1 if c["query_block"] == 1 and rng.random() < 0.5 else _log(rng, 1, 256)
        elif c["query_block"] < 64:
            c["length"] = c["new"] = min(c["length"], max(4096, least))
        c["causal"] = c["paged"] or rng.random() < 0.75
    elif op == "train":
        c["batch"] = _log(rng, 1, 4)
        c["query_block"] = rng.choice([1, 16, 64, 128])
        most = 500000 // (c["batch"] * c["heads"])          # the largest listed case's work
        if c["query_block"] == 1:                           # and room for the plain form's gathered keys
            most = min(most, 16384 // (c["batch"] * c["kv_heads"]))
        c["new"] = c["length"] = _log(rng, 1, min(8192, most))
        c["n_select"] = min(16, max(2, 1024 // c["block"]))
        c["causal"], c["fused"] = rng.random() < 0.75, rng.random() < 0.5
    else:
        c["batch"] = _log(rng, 1, 16)
        c["new"] = rng.choice([1, 1, 4, _log(rng, 1, 512)])
        c["length"] = c["new"] + _log(rng, 1, 16384)
        c["query_block"] = 1 if c["new"] <= 4 else 64
        c["n_select"] = rng.choice([0, 0, 8, 16])
        if c["new"] > 64:
            c["batch"] = min(c["batch"], 2)
    return c


# ------------------------------------------------------------------------------------------------ inputs

def lens_of(c):
    """Tokens held and tokens new of every sequence: the first has the whole length, the others shorter ones."""
    n, new = [], []
    for i in range(c["batch"]):
        f = 1.0 if i == 0 or not c["ragged"] else 0.3 + 0.7 * ((i * 0.6180339887) % 1.0)
        n.append(max(1, int(c["length"] * f)))
        new.append(min(n[-1], max(1, int(c["new"] * f))))
    return n, new


def _lists(c, nqb, nkb, g, device):
    """Seeded lists as a selection leaves them: ascending, the blocks of the queries themselves among them, -1 behind."""
    n, new = lens_of(c)
    B, H, S = c["batch"], c["kv_heads"], c["n_select"]
    n_t = torch.tensor(n, device=device)[:, None, None, None]
    new_t = torch.tensor(new, device=device)[:, None, None, None]
    qb = torch.arange(nqb, device=device)[None, :, None, None]
    kb = torch.arange(nkb, device=device)[None, None, None, :]
    first = n_t - new_t + qb * c["query_block"]
    last = torch.minimum(first + c["query_block"], n_t) - 1
    ok = (kb * c["block"] < n_t) & (qb * c["query_block"] < new_t)
    if c.get("causal", True):
        ok = ok & (kb * c["block"] <= last)
    own_block = (kb >= first // c["block"]) & (kb <= last // c["block"])
    r = torch.rand(B, nqb, H, nkb, generator=g, device=device) + own_block.float() + (kb == 0).float()
    r = torch.where(ok.expand_as(r), r, torch.full_like(r, -1.0))
    take = min(S, nkb)
    val, idx = r.topk(take, dim=-1)
    idx = torch.where(val >= 0, idx, torch.full_like(idx, nkb)).sort(dim=-1).values
    out = torch.full((B, nqb, H, S), -1, dtype=torch.int32, device=device)
    out[..., :take] = torch.where(idx < nkb, idx, torch.full_like(idx, -1)).int()
    return out


def prepare(case, seed):
    c = dict(case)
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    n, new = lens_of(c)
    B, H, HK, D, bs = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["block"]
    T = sum(new)
    s = dict(case=c, max_new=max(new), scale=D ** -0.5)
    s["cu"] = torch.tensor([sum(new[:i]) for i in range(B + 1)], dtype=torch.int32, device=dev)
    s["lengths"] = torch.tensor(n, dtype=torch.int32, device=dev)

    def tokens(heads):
        return torch.randn(T, heads, D, generator=g, device=dev).to(dt)

    if c["op"] == "train" and c["fused"]:
        qkv = torch.randn(T, H + 2 * HK, D, generator=g, device=dev).to(dt)
        q, k, v = qkv[:, :H], qkv[:, H:H + HK], qkv[:, H + HK:]
    else:
        q, k, v = tokens(H), tokens(HK), tokens(HK)
    s["q"] = q
    if c["op"] in ("append", "train") or (c["op"] == "select" and not c["paged"]):
        s["k"], s["v"] = k, v
    if c["op"] == "append" or c["op"] == "attend" or c.get("paged"):
        per = [-(-x // bs) for x in n]
        width, pages = max(per), sum(per) + 3
        perm = torch.randperm(pages, generator=g, device=dev).int()
        table = torch.zeros(B, width, dtype=torch.int32, device=dev)
        at = 0
        for i, p in enumerate(per):
            table[i, :p] = perm[at:at + p]
            at += p
        s["table"] = table
        if c["op"] == "select":
            s["k_pages"] = s["v_pages"] = torch.zeros(pages, HK, bs, D, dtype=dt, device=dev)
            s["key_sums"] = torch.randn(pages, HK, D, generator=g, device=dev) * bs ** 0.5
        else:
            s["k_pages"] = torch.randn(pages, HK, bs, D, generator=g, device=dev, dtype=dt)
            s["v_pages"] = torch.randn(pages, HK, bs, D, generator=g, device=dev, dtype=dt)
            s["key_sums"] = s["k_pages"].double().sum(2).float() if c["op"] == "append" else \
                torch.zeros(pages, HK, D, device=dev)
    if c["op"] == "append" and c["rotary"]:
        i = torch.arange(0, c["rotary"], 2, device=dev, dtype=torch.float64)
        s["inv_freq"] = (10000.0 ** (-i / c["rotary"])).float()
    if c["op"] == "train":
        for x in ("q", "k", "v"):
            s[x] = s[x].detach().requires_grad_()
        s["d_out"] = tokens(H)
    if c["op"] in ("train", "attend") and c["n_select"]:
        s["lists"] = _lists(c, -(-s["max_new"] // c["query_block"]), -(-max(n) // bs), g, dev)
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    return {"append": _append, "select": _select, "train": _train, "attend": _attend}[s["case"]["op"]](s)


def _cache(s):
    """The cache object that a serving program keeps beside its page tensors."""
    if "cache" not in s:
        from cuspamm_b200 import PagedCache
        s["cache"] = PagedCache(s["k_pages"], s["v_pages"], s["key_sums"])
    return s["cache"]


def _padded(x, s, dtype):
    """Packed tokens [T, ...] as [batch, longest, ...] in `dtype`, zeros behind the shorter ones; and who is there."""
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    t = torch.arange(s["max_new"], device=x.device)
    there = t[None, :] < new[:, None]
    at = (s["cu"][:-1, None].long() + t[None, :]).clamp(max=x.shape[0] - 1)
    y = x[at].to(dtype)
    return torch.where(there.view(there.shape + (1,) * (x.dim() - 1)), y, torch.zeros((), dtype=dtype, device=x.device)), there


def _rotated(x, pos, inv_freq, interleaved):
    """x [T, heads, D] turned by pos [T]; the first 2*len(inv_freq) values of each head, in 64-bit angles."""
    r = inv_freq.numel()
    angle = pos.double()[:, None] * inv_freq.double()[None, :]
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    y = x.float()
    a, b = (y[..., 0:2 * r:2], y[..., 1:2 * r:2]) if interleaved else (y[..., :r], y[..., r:2 * r])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, w), dim=-1).flatten(-2) if interleaved else torch.cat((u, w), dim=-1)
    return torch.cat((turned, y[..., 2 * r:]), dim=-1).to(x.dtype)


def _append(s):
    c = s["case"]
    if own:
        q = _cache(s).append(s["k"], s["v"], s["cu"], s["max_new"], s["table"], s["lengths"],
                             inv_freq=s.get("inv_freq"), interleaved=c["interleaved"], q=s["q"])
        return s["k_pages"], s["v_pages"], s["key_sums"], q
    bs, T = c["block"], s["k"].shape[0]
    t = torch.arange(T, device=s["k"].device)
    seq = torch.searchsorted(s["cu"][1:].contiguous(), t.int(), right=True)
    pos = s["lengths"].long()[seq] - (s["cu"][1:].long()[seq] - t)
    k, q = s["k"], s["q"]
    if "inv_freq" in s:
        k = _rotated(k, pos, s["inv_freq"], c["interleaved"])
        q = _rotated(q, pos, s["inv_freq"], c["interleaved"])
    page = s["table"][seq, pos // bs].long()
    s["k_pages"][page, :, pos % bs] = k
    s["v_pages"][page, :, pos % bs] = s["v"]
    # the sums of the touched pages, over the tokens that each holds now
    n = s["lengths"].long()
    first = (n - (s["cu"][1:] - s["cu"][:-1]).long()) // bs
    j = first[:, None] + torch.arange((s["max_new"] + 2 * bs - 2) // bs, device=t.device)
    seq, at = (j * bs < n[:, None]).nonzero(as_tuple=True)
    page = s["table"][seq, j[seq, at]].long()
    there = torch.arange(bs, device=t.device)[None, :] < (n[seq] - j[seq, at] * bs)[:, None]
    s["key_sums"][page] = torch.where(there[:, None, :, None], s["k_pages"][page].double(), 0.0).sum(2).float()
    return s["k_pages"], s["v_pages"], s["key_sums"], q if "inv_freq" in s else q.clone()


def _select(s):
    c = s["case"]
    if own:
        how = dict(query_block=c["query_block"], n_first=c["n_first"], n_local=c["n_local"])
        if c["paged"]:
            return _cache(s).select(s["q"], s["cu"], s["max_new"], s["table"], s["lengths"], c["n_select"], **how)
        from cuspamm_b200 import select_blocks
        return select_blocks(s["q"], s["k"], s["cu"], s["max_new"], c["n_select"], block=c["block"],
                             causal=c["causal"], **how)
    B, HK, D, bs, bq = c["batch"], c["kv_heads"], c["dim"], c["block"], c["query_block"]
    dev = s["q"].device
    n = s["lengths"].long()
    q, _ = _padded(s["q"], s, torch.float64)
    nqb = -(-s["max_new"] // bq)
    q = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, nqb * bq - s["max_new"]))
    q = q.view(B, nqb, bq, HK, -1, D).sum((2, 4))                                  # [B, nqb, HK, D]
    if c["paged"]:
        sums = s["key_sums"][s["table"].long()]                                    # [B, nkb, HK, D]
    else:
        k, _ = _padded(s["k"], s, torch.float64)
        nkb = -(-s["max_new"] // bs)
        k = torch.nn.functional.pad(k, (0, 0, 0, 0, 0, nkb * bs - s["max_new"]))
        sums = k.view(B, nkb, bs, HK, D).sum(2).float()
    nkb = sums.shape[1]
    kb = torch.arange(nkb, device=dev)[None, None, :]
    held = (n[:, None] - torch.arange(nkb, device=dev)[None, :] * bs).clamp(1, bs).double()
    score = torch.einsum("bqhd,bkhd->bhqk", q, sums.double()) / held[:, None, None, :]
    new = (s["cu"][1:] - s["cu"][:-1]).long()[:, None, None]
    qb = torch.arange(nqb, device=dev)[None, :, None]
    first = n[:, None, None] - new + qb * bq
    last = torch.minimum(first + bq, n[:, None, None]) - 1
    ok = (kb * bs < n[:, None, None]) & (qb * bq < new)
    if c["causal"]:
        ok = ok & (kb * bs <= last)
    forced = (kb < c["n_first"]) | ((kb > first // bs - c["n_local"]) & (kb <= last // bs))
    score = torch.where(forced[:, None], torch.inf, score)
    score = torch.where(ok[:, None], score, -torch.inf)
    order = score.sort(dim=-1, descending=True, stable=True)
    take = min(c["n_select"], nkb)
    best, idx = order.values[..., :take], order.indices[..., :take]
    idx = torch.where(best > -torch.inf, idx, nkb).sort(dim=-1).values
    idx = torch.where(idx < nkb, idx, -1)
    idx = torch.nn.functional.pad(idx, (0, c["n_select"] - take), value=-1)
    return idx.permute(0, 2, 1, 3).int().contiguous()


def _listed_keys(s, x, nkb):
    """x [B, longest, HK, D] by blocks, and of those the listed ones: [B, nqb, HK, S*block, D]."""
    c = s["case"]
    B, HK, D, bs = c["batch"], c["kv_heads"], c["dim"], c["block"]
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, nkb * bs - x.shape[1])).view(B, nkb, bs, HK, D)
    x = x.permute(0, 3, 1, 2, 4)                                                   # [B, HK, nkb, bs, D]
    b = torch.arange(B, device=x.device)[:, None, None, None]
    h = torch.arange(HK, device=x.device)[None, None, :, None]
    return x[b, h, s["lists"].long().clamp(min=0)].flatten(3, 4)


def _train(s):
    c = s["case"]
    if own:
        from cuspamm_b200 import block_sparse_attention
        o = block_sparse_attention(s["q"], s["k"], s["v"], s["lists"], s["cu"], s["max_new"], block=c["block"],
                                   query_block=c["query_block"], causal=c["causal"], scale=s["scale"])
        return (o.detach(),) + torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["d_out"])
    with torch.no_grad():
        return _train_plain(s, c)


def _train_plain(s, c):
    B, HK, D, bs, bq = c["batch"], c["kv_heads"], c["dim"], c["block"], c["query_block"]
    dt, dev = s["q"].dtype, s["q"].device
    longest = s["max_new"]
    nqb, nkb = -(-longest // bq), -(-longest // bs)

    def queries(x):
        x, there = _padded(x, s, torch.float32)
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, nqb * bq - longest))
        return x.view(B, nqb, bq, HK, -1, D).permute(0, 1, 3, 2, 4, 5).flatten(3, 4), there   # [B, nqb, HK, bq*G, D]

    q, there = queries(s["q"])
    do, _ = queries(s["d_out"])
    G = q.shape[3] // bq
    kg = _listed_keys(s, _padded(s["k"], s, torch.float32)[0], nkb)
    vg = _listed_keys(s, _padded(s["v"], s, torch.float32)[0], nkb)
    key = (s["lists"].long()[..., None] * bs + torch.arange(bs, device=dev)).flatten(3)        # [B, nqb, HK, S*bs]
    row = (torch.arange(nqb * bq, device=dev).view(nqb, bq, 1).expand(nqb, bq, G)).reshape(1, nqb, 1, bq * G, 1)
    ok = (key >= 0)[..., None, :] & (key < s["lengths"].long()[:, None, None, None])[..., None, :]
    if c["causal"]:
        ok = ok & (key[..., None, :] <= row)
    z = torch.where(ok, q @ kg.transpose(-1, -2) * s["scale"], -torch.inf)
    top = z.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    o = p @ vg
    dp = do @ vg.transpose(-1, -2)
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * s["scale"]
    dq = ds @ kg

    def packed(x, heads):
        """[B, nqb, HK, bq*G, D] back to [T, heads, D]."""
        x = x.view(B, nqb, HK, bq, G, D).permute(0, 1, 3, 2, 4, 5).reshape(B, nqb * bq, heads, D)
        return x[:, :longest][there].to(dt)

    def spread(x):
        """Sums of [B, nqb, HK, S*bs, D] over the query blocks that list a key, as [T, HK, D]."""
        to = torch.zeros(B, HK, nkb * bs, D, device=dev)
        b = torch.arange(B, device=dev)[:, None, None, None].expand_as(key)
        h = torch.arange(HK, device=dev)[None, None, :, None].expand_as(key)
        at = (b * HK + h) * (nkb * bs) + key.clamp(min=0)
        x = torch.where((key >= 0)[..., None], x, 0.0)
        to.view(-1, D).index_add_(0, at.reshape(-1), x.reshape(-1, D))
        return to.permute(0, 2, 1, 3)[:, :longest][there].to(dt)

    return packed(o, s["q"].shape[1]), packed(dq, s["q"].shape[1]), spread(ds.transpose(-1, -2) @ q), \
        spread(p.transpose(-1, -2) @ do)


def _attend(s):
    c = s["case"]
    if own:
        return _cache(s).attend(s["q"], s["cu"], s["max_new"], s["table"], s["lengths"], lists=s.get("lists"),
                                query_block=c["query_block"], scale=s["scale"])
    B, HK, D, bs, bq = c["batch"], c["kv_heads"], c["dim"], c["block"], c["query_block"]
    dev, longest = s["q"].device, s["max_new"]
    n = s["lengths"].long()
    q, there = _padded(s["q"], s, torch.float32)
    pos = n[:, None] - there.sum(1, keepdim=True) + torch.arange(longest, device=dev)          # [B, longest]
    table = s["table"].long()
    if "lists" in s:      # one list for each query block: its pages gathered
        nqb = -(-longest // bq)
        q = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, nqb * bq - longest))
        pos = torch.nn.functional.pad(pos, (0, nqb * bq - longest), value=-1)
        lists = s["lists"].long()
        page = torch.gather(table[:, None, None, :].expand(B, nqb, HK, -1), 3, lists.clamp(min=0))
        h = torch.arange(HK, device=dev)[None, None, :, None]
        kg, vg = s["k_pages"][page, h].flatten(3, 4).float(), s["v_pages"][page, h].flatten(3, 4).float()
        key = (lists[..., None] * bs + torch.arange(bs, device=dev)).flatten(3)                # [B, nqb, HK, S*bs]
    else:                 # every page: one list for all queries
        nqb, bq = 1, longest
        kg = s["k_pages"][table].transpose(1, 2).flatten(2, 3).float()[:, None]                # [B, 1, HK, keys, D]
        vg = s["v_pages"][table].transpose(1, 2).flatten(2, 3).float()[:, None]
        key = torch.arange(kg.shape[3], device=dev)[None, None, None, :]
    q = q.view(B, nqb, bq, HK, -1, D).permute(0, 1, 3, 2, 4, 5).flatten(3, 4)                  # [B, nqb, HK, bq*G, D]
    G = q.shape[3] // bq
    row = pos.view(B, nqb, 1, bq, 1).expand(B, nqb, 1, bq, G).reshape(B, nqb, 1, bq * G, 1)
    ok = (key >= 0)[..., None, :] & (key[..., None, :] <= row)
    z = torch.where(ok, q @ kg.transpose(-1, -2) * s["scale"], -torch.inf)
    top = z.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, p @ torch.where((key >= 0)[..., None], vg, 0.0) / total, 0.0)
    o = o.view(B, nqb, HK, bq, G, D).permute(0, 1, 3, 2, 4, 5).reshape(B, nqb * bq, -1, D)
    return o[:, :longest][there].to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------ work

def work(case):
    c = dict(case)
    n, new = lens_of(c)
    H, HK, D, bs, T = c["heads"], c["kv_heads"], c["dim"], c["block"], sum(new)
    if c["op"] == "append":
        touched = sum((x - 1) // bs - (x - y) // bs + 1 for x, y in zip(n, new))
        old = sum((x - y) % bs for x, y in zip(n, new))            # keys already on the first touched pages
        return {"bytes": 4 * T * HK * D * 2 + 2 * T * H * D * 2 + old * HK * D * 2 + touched * HK * D * 4,
                "flops": 3 * T * (H + HK) * c["rotary"] + T * HK * D}
    if c["op"] == "select":
        nqb = sum(-(-y // c["query_block"]) for y in new)
        nkb = sum(-(-x // bs) for x in n)
        pairs = sum(-(-y // c["query_block"]) * -(-x // bs) for x, y in zip(n, new))
        if c["causal"] and not c["paged"]:
            pairs /= 2
        keys = nkb * HK * D * 4 if c["paged"] else T * HK * D * 2
        return {"bytes": T * H * D * 2 + keys + nqb * HK * c["n_select"] * 4,
                "flops": 2 * pairs * HK * D + T * H * D + (0 if c["paged"] else T * HK * D)}
    most = c["n_select"] * bs if c["n_select"] else 1 << 60
    pairs = keys = 0
    for x, y in zip(n, new):
        if c.get("causal", True):
            lo, hi = x - y + 1, x                                  # keys before and at each of the new tokens
            cut = min(max(most, lo - 1), hi)
            pairs += (lo + cut) * (cut - lo + 1) // 2 + (hi - cut) * most
        else:
            pairs += y * min(most, x)
        keys += x if c["op"] == "train" else min(x, most * -(-y // c["query_block"]))
    if c["op"] == "train":
        return {"bytes": (4 * T * H + 4 * T * HK) * D * 2, "flops": 14 * pairs * H * D}
    return {"bytes": 2 * T * H * D * 2 + 2 * keys * HK * D * 2, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"append": _exact_append, "select": _exact_select, "train": _exact_train,
                "attend": _exact_attend}[case["op"]](s)


def _turn(x, pos, s):
    """x [heads, D] in 64 bits as complex numbers times exp(i * angle)."""
    if "inv_freq" not in s:
        return x
    r = s["inv_freq"].numel()
    unit = torch.polar(torch.ones_like(pos)[:, None] * torch.ones(r, dtype=torch.float64, device=x.device),
                       pos[:, None] * s["inv_freq"].double())[:, None]
    if s["case"]["interleaved"]:
        zc = torch.complex(x[..., 0:2 * r:2].contiguous(), x[..., 1:2 * r:2].contiguous()) * unit
        x[..., 0:2 * r:2], x[..., 1:2 * r:2] = zc.real, zc.imag
    else:
        zc = torch.complex(x[..., :r].contiguous(), x[..., r:2 * r].contiguous()) * unit
        x[..., :r], x[..., r:2 * r] = zc.real, zc.imag
    return x


def _exact_append(s):
    c = s["case"]
    n, new = lens_of(c)
    bs, cu = c["block"], [0]
    kp, vp, ks = s["k_pages"].double(), s["v_pages"].double(), s["key_sums"].double()
    q = s["q"].double()
    for i in range(c["batch"]):
        cu.append(cu[-1] + new[i])
        a, b, p0 = cu[i], cu[i + 1], n[i] - new[i]
        pos = torch.arange(p0, n[i], device=q.device, dtype=torch.float64)
        q[a:b] = _turn(q[a:b].clone(), pos, s)
        k, v = _turn(s["k"][a:b].double(), pos, s), s["v"][a:b].double()
        for j in range(p0 // bs, (n[i] - 1) // bs + 1):
            lo, hi = max(p0, j * bs), min(n[i], (j + 1) * bs)
            page = int(s["table"][i, j])
            kp[page, :, lo - j * bs:hi - j * bs] = k[lo - p0:hi - p0].transpose(0, 1)
            vp[page, :, lo - j * bs:hi - j * bs] = v[lo - p0:hi - p0].transpose(0, 1)
            # the sum is that of the stored, rounded keys: it has no value of its own in 64 bits
    return kp, vp, None, q


def _exact_select(s):
    c = s["case"]
    n, new = lens_of(c)
    B, HK, D, bs, bq, S = c["batch"], c["kv_heads"], c["dim"], c["block"], c["query_block"], c["n_select"]
    dev = s["q"].device
    out = torch.full((B, -(-s["max_new"] // bq), HK, S), -1, dtype=torch.int32, device=dev)
    at = 0
    for i in range(B):
        q = s["q"][at:at + new[i]].double().view(new[i], HK, -1, D).sum(2)
        nqb, nkb = -(-new[i] // bq), -(-n[i] // bs)
        qs = torch.zeros(nqb, HK, D, dtype=torch.float64, device=dev)
        qs.index_add_(0, torch.arange(new[i], device=dev) // bq, q)
        if c["paged"]:
            ks = s["key_sums"][s["table"][i, :nkb].long()].double()
        else:
            ks = torch.zeros(nkb, HK, D, dtype=torch.float64, device=dev)
            ks.index_add_(0, torch.arange(n[i], device=dev) // bs, s["k"][at:at + n[i]].double())
            ks = ks.float().double()
        fill = torch.tensor([min(bs, n[i] - b * bs) for b in range(nkb)], dtype=torch.float64, device=dev)
        first = n[i] - new[i] + torch.arange(nqb, device=dev) * bq
        last = torch.clamp(first + bq, max=n[i]) - 1
        b = torch.arange(nkb, device=dev)
        for h in range(HK):
            score = (qs[:, h] @ ks[:, h].T) / fill
            must = (b < c["n_first"])[None] | ((b[None] > (first // bs)[:, None] - c["n_local"]) & (b[None] <= (last // bs)[:, None]))
            score[must] = torch.inf
            if c["causal"]:
                score[b[None] * bs > last[:, None]] = -torch.inf
            take = min(S, nkb)
            rank = score.argsort(dim=1, descending=True, stable=True)[:, :take]
            keep = torch.zeros_like(score, dtype=torch.bool).scatter_(1, rank, True) & (score > -torch.inf)
            place = keep.long().cumsum(1) - 1
            r, col = keep.nonzero(as_tuple=True)
            out[i, :nqb, h][r, place[r, col]] = col.int()
        at += new[i]
    return out


def _exact_train(s):
    c = s["case"]
    _, new = lens_of(c)
    H, HK, D, bs, bq = c["heads"], c["kv_heads"], c["dim"], c["block"], c["query_block"]
    if sum(x * x for x in new) * H > 8e9:
        return None
    G, dev, at = H // HK, s["q"].device, 0
    grads = [torch.zeros(s[x].shape, dtype=torch.float64, device=dev) for x in ("q", "q", "k", "v")]
    for i, x in enumerate(new):
        t = torch.arange(x, device=dev)
        for h in range(HK):
            rows = s["lists"][i, t // bq, h].long()                                # [x, S]
            on = torch.zeros(x, -(-x // bs) + 1, dtype=torch.bool, device=dev)
            on.scatter_(1, torch.where(rows < 0, on.shape[1] - 1, rows), True)
            on = on[:, t // bs]
            if c["causal"]:
                on = on & (t[None, :] <= t[:, None])
            k, v = s["k"][at:at + x, h].double(), s["v"][at:at + x, h].double()
            for j in range(h * G, (h + 1) * G):
                q, do = s["q"][at:at + x, j].double(), s["d_out"][at:at + x, j].double()
                p = torch.softmax((q @ k.T * s["scale"]).masked_fill(~on, -torch.inf), dim=1).nan_to_num(0.0)
                o = p @ v
                ds = p * (do @ v.T - (do * o).sum(1, keepdim=True)) * s["scale"]
                grads[0][at:at + x, j], grads[1][at:at + x, j] = o, ds @ k
                grads[2][at:at + x, h] += ds.T @ q
                grads[3][at:at + x, h] += p.T @ do
        at += x
    return tuple(grads)


def _exact_attend(s):
    c = s["case"]
    n, new = lens_of(c)
    H, HK, D, bs, bq = c["heads"], c["kv_heads"], c["dim"], c["block"], c["query_block"]
    G, dev, at = H // HK, s["q"].device, 0
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    for i in range(c["batch"]):
        nkb = -(-n[i] // bs)
        page = s["table"][i, :nkb].long()
        t = torch.arange(new[i], device=dev)
        reach = torch.arange(n[i], device=dev)[None, :] <= (n[i] - new[i] + t)[:, None]
        for h in range(HK):
            k = s["k_pages"][page, h].flatten(0, 1)[:n[i]].double()
            v = s["v_pages"][page, h].flatten(0, 1)[:n[i]].double()
            on = reach
            if "lists" in s:
                rows = s["lists"][i, t // bq, h].long()
                some = torch.zeros(new[i], nkb + 1, dtype=torch.bool, device=dev)
                some.scatter_(1, torch.where(rows < 0, nkb, rows), True)
                on = reach & some[:, torch.arange(n[i], device=dev) // bs]
            for j in range(h * G, (h + 1) * G):
                z = (s["q"][at:at + new[i], j].double() @ k.T * s["scale"]).masked_fill(~on, -torch.inf)
                out[at:at + new[i], j] = torch.softmax(z, dim=1).nan_to_num(0.0) @ v
        at += new[i]
    return out
