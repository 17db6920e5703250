"""The attention operators on the GPU against their plain 64-bit forms; bounds as derived in _attention_plain.py."""
import numpy as np
import pytest
import torch

import _attention_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


def tokens(g, n, heads, dim, dtype):
    return torch.randn(n, heads, dim, generator=g).to(dtype).to(DEV)


def cu_of(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)


def random_lists(g, lens, held, kv_heads, block, query_block, n_select, causal, junk=False):
    """Lists with the queries' own blocks and random others; with `junk` also entries that have to be skipped."""
    nqb = max(1, -(-max(lens) // query_block))
    out = torch.full((len(lens), nqb, kv_heads, n_select), -1, dtype=torch.int32)
    for s, (n, k) in enumerate(zip(lens, held)):
        for i in range(-(-n // query_block)):
            last = k - n + min((i + 1) * query_block, n) - 1
            blocks = (last // block + 1) if causal else -(-k // block)
            for h in range(kv_heads):
                pick = torch.randperm(blocks, generator=g)[:n_select].sort().values.int()
                out[s, i, h, :len(pick)] = pick
    if junk:
        out[..., 1::4] = torch.randint(-5, 40, out[..., 1::4].shape, generator=g).int()
        out[0, 0] = -1                                            # a query block that reads nothing
    return out.to(DEV)


def expect(q, k, v, lists, lens, block, query_block, causal, scale, d_o=None):
    """Values and bounds of packed self attention, all heads."""
    H, HK = q.shape[1], k.shape[1]
    names = ("o", "lse") + (("dq", "dk", "dv") if d_o is not None else ())
    shapes = dict(o=q.shape, lse=q.shape[:2], dq=q.shape, dk=k.shape, dv=v.shape)
    val = {n: torch.zeros(shapes[n], dtype=torch.float64, device=DEV) for n in names}
    tol = {n: torch.zeros(shapes[n], dtype=torch.float64, device=DEV) for n in names}
    at = 0
    for s, n in enumerate(lens):
        r = slice(at, at + n)
        for h in range(H):
            hk = h // (H // HK)
            ok = plain.mask_of(lists[s].cpu(), n, n, 0, block, query_block, causal, hk).to(DEV)
            x, t = plain.attend(q[r, h], k[r, hk], v[r, hk], ok, scale, d_o[r, h] if d_o is not None else None)
            for name in names:
                to = hk if name in ("dk", "dv") else h
                val[name][r, to] += x[name]
                tol[name][r, to] += t[name]
        at += n
    val["lse"][at:] = -torch.inf
    return val, tol


def near(got, want, bound, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), f"{what}: infinities"
    off = (got[~inf] - want[~inf]).abs() - bound[~inf]
    assert not bool(torch.isnan(got).any()), f"{what}: NaN"
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max()):.3g} over the bound"


CASES = [
    # lens, heads, kv_heads, dim, dtype, block, query_block, n_select, causal
    ([130, 1, 0, 257], 4, 2, 64, BF, 64, 64, 3, True),
    ([200], 16, 1, 128, HF, 64, 1, 2, True),
    ([129, 63], 3, 1, 128, BF, 32, 16, 5, True),
    ([300], 6, 2, 64, HF, 16, 128, 9, False),
    ([257, 5], 2, 2, 128, BF, 128, 128, 2, True),
    ([1], 1, 1, 64, BF, 16, 1, 1, True),
    ([70, 190], 5, 1, 64, HF, 16, 7, 6, True),
    ([333], 8, 2, 128, HF, 128, 48, 2, False),
    ([640], 4, 1, 128, BF, 64, 64, 4, True),
    ([150], 40, 1, 64, BF, 32, 1, 3, True),
    ([384, 100], 4, 4, 64, BF, 64, 1000, 6, True),
]


@pytest.mark.parametrize("case", CASES, ids=[f"{i}" for i in range(len(CASES))])
@pytest.mark.parametrize("junk", [False, True])
def test_sparse_attention_and_its_gradients(case, junk):
    from cuspamm_b200 import block_sparse_attention

    lens, H, HK, D, dt, block, qb, n_select, causal = case
    g = torch.Generator().manual_seed(len(lens) * 1000 + H * 10 + D)
    T = sum(lens)
    q, k, v, d_o = (tokens(g, T, n, D, dt) for n in (H, HK, HK, H))
    lists = random_lists(g, lens, lens, HK, block, qb, n_select, causal, junk)
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    o, lse = block_sparse_attention(*x, lists, cu_of(lens), max(lens), block=block, query_block=qb, causal=causal, return_lse=True)
    dq, dk, dv = torch.autograd.grad(o, x, d_o)
    val, tol = expect(q, k, v, lists, lens, block, qb, causal, D ** -0.5, d_o)
    got = dict(o=o.detach(), lse=lse, dq=dq, dk=dk, dv=dv)
    for n in got:
        near(got[n], val[n], tol[n], n)


def test_gradients_against_differences():
    """The gradient along a direction against differences of the 64-bit formula."""
    from cuspamm_b200 import block_sparse_attention

    g = torch.Generator().manual_seed(5)
    lens, H, HK, D, block, qb = [90], 4, 2, 64, 16, 8
    q, k, v, d_o = (tokens(g, 90, n, D, HF) for n in (H, HK, HK, H))
    lists = random_lists(g, lens, lens, HK, block, qb, 3, True)
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    o = block_sparse_attention(*x, lists, cu_of(lens), 90, block=block, query_block=qb)
    grads = torch.autograd.grad(o, x, d_o)
    _, tol = expect(q, k, v, lists, lens, block, qb, True, D ** -0.5, d_o)
    masks = [plain.mask_of(lists[0].cpu(), 90, 90, 0, block, qb, True, h).to(DEV) for h in range(HK)]

    def loss(q, k, v):
        total = 0.0
        for h in range(H):
            z = (q[:, h] @ k[:, h // 2].T * D ** -0.5).masked_fill(~masks[h // 2], -torch.inf)
            p = torch.exp(z - z.amax(1, keepdim=True).nan_to_num(neginf=0.0))
            o = p @ v[:, h // 2] / p.sum(1, keepdim=True).clamp(min=1e-300)
            total += float((o * d_o[:, h].double()).sum())
        return total

    for i, name in enumerate(("dq", "dk", "dv")):
        for trial in range(3):
            d = torch.randn(x[i].shape, generator=g, dtype=torch.float64).to(DEV)
            at = [t.double() for t in (q, k, v)]
            h = 1e-5
            up, down = list(at), list(at)
            up[i], down[i] = at[i] + h * d, at[i] - h * d
            want = (loss(*up) - loss(*down)) / (2 * h)
            got = float((grads[i].double() * d).sum())
            # every element off by at most its bound; 1e-6 for the differences themselves
            assert abs(got - want) <= float((tol[name] * d.abs()).sum()) + 1e-6 * max(1.0, abs(want)), name


def test_same_bits_twice_and_on_another_stream():
    from cuspamm_b200 import block_sparse_attention

    g = torch.Generator().manual_seed(3)
    lens = [700, 333]
    q, k, v, d_o = (tokens(g, 1033, n, 128, BF) for n in (8, 2, 2, 8))
    lists = random_lists(g, lens, lens, 2, 64, 16, 4, True)
    cu = cu_of(lens)

    def once():
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        o = block_sparse_attention(*x, lists, cu, 700, query_block=16)
        return (o.detach(),) + torch.autograd.grad(o, x, d_o)

    a = once()
    stream = torch.cuda.Stream(DEV)
    stream.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(stream):
        b = once()
    torch.cuda.current_stream(DEV).wait_stream(stream)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_views_expanded_heads_and_padding_rows():
    """q, k, v cut from one tensor, keys expanded over heads, an expanded output gradient, rows behind the last sequence."""
    from cuspamm_b200 import block_sparse_attention

    g = torch.Generator().manual_seed(11)
    lens, T, H, D = [100, 41], 160, 4, 64
    fused = tokens(g, T, H + 2, D, BF)
    lists = random_lists(g, lens, lens, 4, 16, 32, 4, True)
    f = fused.clone().requires_grad_()
    q, k, v = f[:, :H], f[:, H:H + 1].expand(T, 4, D), f[:, H + 1:].expand(T, 4, D)
    o = block_sparse_attention(q, k, v, lists, cu_of(lens), 100, block=16, query_block=32)
    assert not bool(o[141:].any())
    (df,) = torch.autograd.grad(o.float().sum(), f)
    one = torch.ones(T, H, D, dtype=BF, device=DEV)
    val, tol = expect(fused[:, :H], k.detach(), v.detach(), lists, lens, 16, 32, True, D ** -0.5, one)
    near(o.detach(), val["o"], tol["o"], "o")
    near(df[:, :H], val["dq"], tol["dq"], "dq")
    u = plain.half_step(BF)
    for i, n in ((H, "dk"), (H + 1, "dv")):
        want = val[n].sum(1)
        # four rounded gradients are added in bf16 or float: three more roundings of at most the sum of magnitudes
        bound = tol[n].sum(1) + 4 * u * (val[n].abs() + tol[n]).sum(1)
        near(df[:, i], want, bound, n)


def test_nothing_to_do():
    from cuspamm_b200 import PagedCache, block_sparse_attention, select_blocks

    e = lambda n, h: torch.zeros(n, h, 64, dtype=BF, device=DEV)  # noqa: E731
    for lens, T in (([0, 0], 0), ([], 0), ([0], 7)):
        cu = cu_of(lens)
        lists = select_blocks(e(T, 2), e(T, 1), cu, 0, 4)
        assert lists.shape == (len(lens), 0, 1, 4)
        q = torch.ones(T, 2, 64, dtype=BF, device=DEV).requires_grad_()
        o = block_sparse_attention(q, e(T, 1), e(T, 1), lists, cu, 0)
        assert o.shape == q.shape and not bool(o.any())
        if T:
            (dq,) = torch.autograd.grad(o, q, torch.ones_like(o))
            assert not bool(dq.any())
    cache = PagedCache.empty(2, 1, 64, page_size=16, device=DEV)
    table, held = torch.zeros(1, 0, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    o = cache.attend(torch.ones(3, 2, 64, dtype=BF, device=DEV), cu_of([0]), 1, table, held)
    assert not bool(o.any())
    cache.check()


# ------------------------------------------------------------------------------------------------ the cache

def build_cache(g, held, kv_heads, dim, dtype, page, spare=2, nan_behind=True):
    """A cache with random pages in random order; what lies behind a sequence's last key is NaN."""
    per = [-(-n // page) for n in held]
    pages, width = sum(per) + spare, max(1, max(per))
    k, v = (torch.randn(pages, kv_heads, page, dim, generator=g).to(dtype) for _ in range(2))
    perm = torch.randperm(pages, generator=g).int()
    table = torch.full((len(held), width), 2 ** 30, dtype=torch.int32)          # never read behind the length
    at = 0
    for s, p in enumerate(per):
        table[s, :p] = perm[at:at + p]
        at += p
        if nan_behind and held[s] % page:
            k[table[s, p - 1], :, held[s] % page:] = torch.nan
            v[table[s, p - 1], :, held[s] % page:] = torch.nan
    return k.to(DEV), v.to(DEV), table.to(DEV), torch.tensor(held, dtype=torch.int32, device=DEV)


def flat(pages, table, s, n, h):
    page = pages.shape[2]
    return pages[table[s, :-(-n // page)].long(), h].flatten(0, 1)[:n]


PAGED = [
    # held, new, heads, kv_heads, dim, dtype, page, query_block, n_select
    ([65], [1], 8, 2, 64, BF, 64, 1, 0),
    ([1, 700, 16], [1, 1, 1], 16, 1, 128, BF, 16, 1, 0),
    ([5000, 333], [1, 1], 4, 4, 128, HF, 128, 1, 0),
    ([300, 40, 129], [70, 40, 1], 6, 2, 64, HF, 32, 16, 0),
    ([900, 200], [4, 3], 8, 1, 128, BF, 64, 1, 5),
    ([513, 77], [200, 77], 12, 4, 128, HF, 64, 64, 3),
    ([2049], [129], 5, 1, 64, BF, 16, 128, 20),
    ([3, 2], [5, 2], 2, 1, 64, BF, 16, 1, 0),                    # more new tokens than the length holds: empty rows
    ([1500], [300], 8, 2, 128, BF, 64, 64, 0),
]


@pytest.mark.parametrize("case", PAGED, ids=[f"{i}" for i in range(len(PAGED))])
def test_attend_over_pages(case):
    from cuspamm_b200 import PagedCache

    held, new, H, HK, D, dt, page, qb, n_select = case
    g = torch.Generator().manual_seed(sum(held))
    k, v, table, lengths = build_cache(g, held, HK, D, dt, page)
    q = tokens(g, sum(new) + 2, H, D, dt)
    cache = PagedCache(k, v)
    lists = random_lists(g, new, held, HK, page, qb, n_select, True, junk=True) if n_select else None
    out = torch.full_like(q, 7.0)
    o, lse = cache.attend(q, cu_of(new), max(new), table, lengths, lists=lists, query_block=qb, out=out, return_lse=True)
    assert o is out and bool((out[sum(new):] == 7.0).all())
    again = cache.attend(q, cu_of(new), max(new), table, lengths, lists=lists, query_block=qb)
    assert torch.equal(again[:sum(new)], out[:sum(new)]) and not bool(again[sum(new):].any())
    at = 0
    for s, (n, m) in enumerate(zip(held, new)):
        for h in range(H):
            hk = h // (H // HK)
            ok = plain.mask_of(None if lists is None else lists[s].cpu(), m, n, n - m, page, qb, True, hk).to(DEV)
            val, tol = plain.attend(q[at:at + m, h], flat(k, table, s, n, hk), flat(v, table, s, n, hk), ok, D ** -0.5)
            near(o[at:at + m, h], val["o"], tol["o"], f"o {s} {h}")
            near(lse[at:at + m, h], val["lse"], tol["lse"], f"lse {s} {h}")
        at += m
    cache.check()


def test_bad_pages_and_lengths_are_masked_and_reported():
    from cuspamm_b200 import PagedCache, SpammError

    g = torch.Generator().manual_seed(2)
    held, page = [100, 50], 16
    k, v, table, lengths = build_cache(g, held, 1, 64, BF, page)
    q, cu = tokens(g, 2, 2, 64, BF), cu_of([1, 1])
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        cache = PagedCache(k, v)
        t = table.clone()
        t[0, 2] = bad
        o = cache.attend(q, cu, 1, t, lengths)
        for h in range(2):
            ok = torch.ones(1, 100, dtype=torch.bool, device=DEV)
            ok[0, 32:48] = False
            kk, vv = flat(k, table, 0, 100, 0), flat(v, table, 0, 100, 0)
            val, tol = plain.attend(q[:1, h], kk, vv, ok, 64 ** -0.5)
            near(o[:1, h], val["o"], tol["o"], "o")
        with pytest.raises(SpammError):
            cache.check()
        cache.check()                                             # reported once
        before = cache.k.clone()
        new = tokens(g, 2, 1, 64, BF)
        t[0, 6] = bad
        cache.append(new, new, cu, 1, t, lengths)
        last = table[1, 3].item()
        rest = [p for p in range(k.shape[0]) if p != last]
        assert torch.equal(cache.k[rest].nan_to_num(), before[rest].nan_to_num())
        with pytest.raises(SpammError):
            cache.check()
    cache = PagedCache(k, v)
    cache.attend(q, cu, 1, table[:, :2].contiguous(), torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device=DEV))
    with pytest.raises(SpammError):
        cache.check()
    cache.attend(q, cu_of([2, 0]), 1, table, lengths)             # more new tokens than max_new
    with pytest.raises(SpammError):
        cache.check()


APPENDS = [
    # held after, new, heads, kv_heads, dim, dtype, page, n_freq, interleaved
    ([1], [1], 2, 1, 64, BF, 16, 32, False),
    ([65, 64, 1000, 7], [1, 1, 1, 1], 8, 2, 128, BF, 64, 64, False),
    ([300, 17, 128], [300, 1, 70], 6, 3, 128, HF, 32, 32, True),
    ([100000, 50], [130, 33], 4, 4, 64, HF, 128, 16, False),
    ([77, 0, 40], [50, 0, 40], 3, 1, 64, BF, 16, 0, False),
    ([40], [40], 32, 16, 128, BF, 16, 8, True),
]


@pytest.mark.parametrize("case", APPENDS, ids=[f"{i}" for i in range(len(APPENDS))])
def test_append(case):
    from cuspamm_b200 import PagedCache

    held, new, H, HK, D, dt, page, n_freq, inter = case
    g = torch.Generator().manual_seed(sum(held) + n_freq)
    k, v, table, lengths = build_cache(g, held, HK, D, dt, page, nan_behind=False)
    T = sum(new)
    fused = tokens(g, T + 1, H + 2 * HK, D, dt)
    q, nk, nv = fused[:, :H], fused[:, H:H + HK], fused[:, H + HK:]
    inv = (1e4 ** (-torch.arange(n_freq, dtype=torch.float64) / max(1, n_freq))).float().to(DEV) if n_freq else None
    cache = PagedCache(k.clone(), v.clone())
    cache.key_sums.fill_(5.0)
    rq = cache.append(nk, nv, cu_of(new), max(new), table, lengths, inv_freq=inv, interleaved=inter, q=q)
    want_k, want_v, want_s = k.clone(), v.clone(), torch.full_like(cache.key_sums, 5.0)
    want_q = torch.zeros(q.shape, dtype=dt, device=DEV)
    at = 0
    for s, (n, m) in enumerate(zip(held, new)):
        pos = torch.arange(n - m, n, device=DEV)
        turn = (lambda x: plain.rotate(x, pos, inv, inter)) if n_freq else (lambda x: x)
        want_q[at:at + m] = turn(q[at:at + m])
        rk = turn(nk[at:at + m])
        for i in range(m):
            p = table[s, (n - m + i) // page].long()
            want_k[p, :, (n - m + i) % page] = rk[i]
            want_v[p, :, (n - m + i) % page] = nv[at + i]
        for b in range((n - m) // page, -(-n // page) if m else 0):
            p = table[s, b].long()
            want_s[p] = want_k[p, :, :min(page, n - b * page)].double().sum(1).float()
        at += m
    # cosines and sines are 64-bit ones rounded to float and everything after them is rounded step by step: equal
    assert torch.equal(cache.v, want_v)
    assert torch.equal(cache.k, want_k)
    assert torch.equal(rq, want_q)
    assert torch.equal(cache.key_sums, want_s)
    cache.check()


SELECT = [
    # lens, heads, kv_heads, dim, dtype, block, query_block, n_select, n_first, n_local, causal
    ([1000, 1, 0, 257], 4, 2, 64, BF, 16, 16, 7, 1, 2, True),
    ([640], 16, 2, 128, HF, 32, 1, 5, 1, 2, True),
    ([900, 100], 6, 3, 128, BF, 64, 64, 4, 0, 1, True),
    ([777], 2, 2, 64, HF, 16, 128, 12, 0, 0, False),
    ([500], 3, 1, 128, BF, 128, 100, 3, 0, 1, True),
    ([300], 4, 4, 64, BF, 16, 7, 19, 1, 0, True),
]


@pytest.mark.parametrize("case", SELECT, ids=[f"{i}" for i in range(len(SELECT))])
@pytest.mark.parametrize("paged", [False, True])
def test_select(case, paged):
    from cuspamm_b200 import PagedCache, select_blocks

    lens, H, HK, D, dt, block, qb, n_select, n_first, n_local, causal = case
    if paged and not causal:
        pytest.skip("the cache is read causally")
    g = torch.Generator().manual_seed(sum(lens) + D)
    T = sum(lens)
    if paged:
        new = [max(1, n // 3) if n else 0 for n in lens]
        k, v, table, lengths = build_cache(g, lens, HK, D, dt, block)
        cache = PagedCache(k, v)
        cache.key_sums.copy_(torch.randn(cache.key_sums.shape, generator=g))
        q = tokens(g, sum(new), H, D, dt)
        got = cache.select(q, cu_of(new), max(new), table, lengths, n_select, query_block=qb, n_first=n_first, n_local=n_local)
        cache.check()
    else:
        new = lens
        q, k = tokens(g, T, H, D, dt), tokens(g, T, HK, D, dt)
        got = select_blocks(q, k, cu_of(lens), max(lens), n_select, block=block, query_block=qb, n_first=n_first,
                            n_local=n_local, causal=causal)
    want = torch.full(got.shape, -1, dtype=torch.int32)
    at = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        nb = -(-n // block)
        if paged:
            sums = cache.key_sums[table[s, :nb].long()].cpu()
        else:
            sums = torch.stack([k[at + b * block:min(at + (b + 1) * block, at + n)].double().sum(0).float() for b in range(nb)]).cpu() \
                if nb else torch.zeros(0, HK, D)
        held = torch.tensor([min(block, n - b * block) for b in range(nb)])
        x = plain.lists_of(q[at:at + m].cpu(), sums, held, n, n - m, block, qb, n_select, n_first, n_local, causal)
        want[s, :x.shape[0]] = x
        at += m
    assert torch.equal(got.cpu(), want)


def test_select_ties_zeros_infinities_and_nan():
    """Equal scores go to the lower block; infinite ones rank by their sign, NaN behind them."""
    from cuspamm_b200 import PagedCache

    held, page, nb = [1600], 16, 100
    cache = PagedCache.empty(100, 1, 64, page_size=page, device=DEV)
    table = torch.arange(100, dtype=torch.int32, device=DEV)[None]
    lengths = torch.tensor(held, dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 1, 64, dtype=BF, device=DEV)
    q[0, 0, 0] = 1.0
    cu = cu_of([1])
    pick = lambda n, **kw: cache.select(q, cu, 1, table, lengths, n, **{"n_first": 0, "n_local": 0, **kw})[0, 0, 0].tolist()  # noqa: E731
    assert pick(5) == [0, 1, 2, 3, 4]                             # all zero
    cache.key_sums[:, 0, 0] = torch.tensor([1.0, -0.0] * 50, device=DEV)
    cache.key_sums[1::4, 0, 0] = 0.0
    assert pick(53) == sorted(list(range(0, 100, 2)) + [1, 3, 5])
    cache.key_sums[7, 0, 0], cache.key_sums[9, 0, 0], cache.key_sums[11, 0, 0] = torch.inf, torch.nan, -torch.inf
    assert pick(1) == [7]
    assert pick(98) == [b for b in range(100) if b not in (9, 11)]
    assert pick(99) == [b for b in range(100) if b != 9]
    assert pick(100) == list(range(100))
    assert pick(3, n_first=1, n_local=1) == [0, 7, 99]


# ------------------------------------------------------------------------------------------------ together

def test_serving_run_prompts_steps_rollback():
    """Prompts in chunks, then single tokens, with a rollback: append, select and attend in turn, each step against the
    plain form over the whole history."""
    from cuspamm_b200 import PagedCache

    g = torch.Generator().manual_seed(21)
    H, HK, D, page, dt = 8, 2, 64, 16, BF
    inv = (1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().to(DEV)
    cache = PagedCache.empty(64, HK, D, page_size=page, dtype=dt, device=DEV)
    perm = torch.randperm(64, generator=g).int().to(DEV)
    table = torch.stack([perm[:20], perm[20:40]]).contiguous()
    hist_k, hist_v = [torch.zeros(0, HK, D, dtype=dt, device=DEV)] * 2, [torch.zeros(0, HK, D, dtype=dt, device=DEV)] * 2
    steps = [([100, 37], None), ([90, 1], None), ([1, 1], None), ([5, 0], None), ([1, 1], [4, 0]), ([3, 64], None)]
    for step, (new, back) in enumerate(steps):
        if back:                                                  # the last tokens of a sequence are dropped again
            hist_k = [x[:len(x) - b] for x, b in zip(hist_k, back)]
            hist_v = [x[:len(x) - b] for x, b in zip(hist_v, back)]
        cu, T = cu_of(new), sum(new)
        q, k, v = tokens(g, T, H, D, dt), tokens(g, T, HK, D, dt), tokens(g, T, HK, D, dt)
        at = [0, new[0]]
        hist_rk = []
        for s in range(2):
            r = slice(at[s], at[s] + new[s])
            pos = torch.arange(len(hist_k[s]), len(hist_k[s]) + new[s], device=DEV)
            hist_k[s] = torch.cat([hist_k[s], plain.rotate(k[r], pos, inv, False)])
            hist_v[s] = torch.cat([hist_v[s], v[r]])
            hist_rk.append(plain.rotate(q[r], pos, inv, False))
        held = [len(x) for x in hist_k]
        lengths = torch.tensor(held, dtype=torch.int32, device=DEV)
        rq = cache.append(k, v, cu, max(new), table, lengths, inv_freq=inv, q=q)
        assert torch.equal(rq, torch.cat(hist_rk))
        qb = 16 if max(new) > 1 else 1
        lists = cache.select(rq, cu, max(new), table, lengths, 6, query_block=qb, n_first=1, n_local=2)
        for use in (lists, None):
            o = cache.attend(rq, cu, max(new), table, lengths, lists=use, query_block=qb)
            for s in range(2):
                n, m = held[s], new[s]
                nb = -(-n // page)
                sums = torch.stack([hist_k[s][b * page:(b + 1) * page].double().sum(0).float() for b in range(nb)]).cpu()
                fill = torch.tensor([min(page, n - b * page) for b in range(nb)])
                x = plain.lists_of(rq[at[s]:at[s] + m].cpu(), sums, fill, n, n - m, page, qb, 6, 1, 2, True)
                assert torch.equal(lists[s, :x.shape[0]].cpu(), x)
                for h in range(H):
                    ok = plain.mask_of(None if use is None else x, m, n, n - m, page, qb, True, h // 4).to(DEV)
                    val, tol = plain.attend(rq[at[s]:at[s] + m, h], hist_k[s][:, h // 4], hist_v[s][:, h // 4], ok, D ** -0.5)
                    near(o[at[s]:at[s] + m, h], val["o"], tol["o"], f"step {step}")
    cache.check()


def test_training_run_select_then_attend():
    from cuspamm_b200 import block_sparse_attention, select_blocks

    g = torch.Generator().manual_seed(31)
    lens, H, HK, D = [400, 150], 8, 2, 128
    q, k, v, d_o = (tokens(g, 550, n, D, HF) for n in (H, HK, HK, H))
    cu = cu_of(lens)
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    lists = select_blocks(x[0], x[1], cu, 400, 4, block=32, query_block=32, n_first=1, n_local=1)
    o = block_sparse_attention(*x, lists, cu, 400, block=32, query_block=32)
    o.backward(d_o)
    val, tol = expect(q, k, v, lists, lens, 32, 32, True, D ** -0.5, d_o)
    for n, got in (("o", o.detach()), ("dq", x[0].grad), ("dk", x[1].grad), ("dv", x[2].grad)):
        near(got, val[n], tol[n], n)


def test_captured_steps_replay_on_new_inputs():
    """Two decoding graphs of one cache, replayed in turn while the tables, lengths and tokens change under them."""
    from cuspamm_b200 import PagedCache

    g = torch.Generator().manual_seed(41)
    H, HK, D, page = 8, 2, 128, 64
    held = [1000, 2500]
    k, v, table, lengths = build_cache(g, held, HK, D, BF, page, spare=4, nan_behind=False)
    cache, eager = PagedCache(k.clone(), v.clone()), PagedCache(k.clone(), v.clone())
    for c in (cache, eager):
        c.key_sums.copy_(c.k.double().sum(2).float())
    cu, inv = cu_of([1, 1]), torch.ones(64, device=DEV) * 0.01
    bufs = [tuple(tokens(g, 2, n, D, BF) for n in (H, HK, HK)) for _ in range(2)]

    def step(c, q, k, v, lens):
        rq = c.append(k, v, cu, 1, table, lens, inv_freq=inv, q=q)
        lists = c.select(rq, cu, 1, table, lens, 8)
        return c.attend(rq, cu, 1, table, lens, lists=lists), c.attend(rq, cu, 1, table, lens), lists

    step(cache, *bufs[0], lengths)
    torch.cuda.synchronize()
    graphs = []
    for b in bufs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cache, *b, lengths)
        graphs.append((graph, out))
    for i in range(6):
        lengths += 1 if i else 0
        b, (graph, out) = bufs[i % 2], graphs[i % 2]
        for x in b:
            x.copy_(torch.randn(x.shape, generator=g))
        want = step(eager, *b, lengths)
        graph.replay()
        for x, y in zip(out, want):
            assert torch.equal(x, y)
    assert torch.equal(cache.k, eager.k) and torch.equal(cache.key_sums, eager.key_sums)
    cache.check()


def test_captured_training_step():
    from cuspamm_b200 import block_sparse_attention, select_blocks

    g = torch.Generator().manual_seed(51)
    cu = cu_of([300])
    q, k, v, d_o = (tokens(g, 300, n, 64, BF) for n in (4, 2, 2, 4))
    x = [t.clone().requires_grad_() for t in (q, k, v)]

    def step():
        lists = select_blocks(x[0], x[1], cu, 300, 3, n_first=0)
        o = block_sparse_attention(*x, lists, cu, 300)
        return (o.detach(),) + torch.autograd.grad(o, x, d_o)

    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(DEV).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        with torch.no_grad():
            for t in x:
                t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("lens,H,HK,qb,block", [([700], 4, 4, 1, 16), ([5000], 2, 2, 4, 16), ([2100, 900], 8, 4, 2, 16),
                                                ([17000], 1, 1, 8, 16)])
def test_select_many_lists(lens, H, HK, qb, block):
    """Enough lists for the kernels that work on tiles of them, and on single ones over many blocks; infinities and NaN among
    the queries and keys."""
    from cuspamm_b200 import select_blocks

    g = torch.Generator().manual_seed(len(lens) + lens[0])
    T, D = sum(lens), 64
    q, k = tokens(g, T, H, D, BF), tokens(g, T, HK, D, BF)
    k[5, 0, 3], k[40, 0, 7], k[90, HK - 1, 1] = torch.inf, -torch.inf, torch.nan
    q[60, 0, 2], q[200, H - 1, 9] = torch.inf, torch.nan
    got = select_blocks(q, k, cu_of(lens), max(lens), 8, block=block, query_block=qb, n_first=1, n_local=2).cpu()
    at = 0
    for s, n in enumerate(lens):
        nb = -(-n // block)
        sums = torch.stack([k[at + b * block:min(at + (b + 1) * block, at + n)].double().sum(0).float() for b in range(nb)]).double()
        held = torch.tensor([min(block, n - b * block) for b in range(nb)], device=DEV).double()
        qs = q[at:at + n].double().view(n, HK, H // HK, D).sum(2)
        nqb = -(-n // qb)
        qs = torch.zeros(nqb, HK, D, dtype=torch.float64, device=DEV).index_add_(0, torch.arange(n, device=DEV) // qb, qs)
        first = torch.arange(nqb, device=DEV) * qb
        last = torch.clamp(first + qb, max=n) - 1
        b = torch.arange(nb, device=DEV)
        for h in range(HK):
            # the products one by one: infinities times zero and against each other must be NaN in every order of summation
            score = torch.stack([(x[None] * sums[:, h]).sum(1) for x in qs[:, h]]) / held
            rank = torch.where(torch.isnan(score), -torch.inf, score)
            nan = torch.isnan(score)
            forced = (b < 1)[None] | ((b > (first // block)[:, None] - 2) & (b <= (last // block)[:, None]))
            ok = b[None] * block <= last[:, None]
            # by rank: forced, then by score, NaN behind minus infinity, then by index; not candidates last
            key = torch.where(forced, torch.inf, rank)
            level = torch.where(ok, torch.where(forced, 3, torch.where(nan, 1, 2)), 0)
            by = torch.argsort(key, dim=1, descending=True, stable=True)
            by = torch.gather(by, 1, torch.argsort(torch.gather(level, 1, by), dim=1, descending=True, stable=True))[:, :8]
            pick = torch.where(torch.gather(level, 1, by) > 0, by, nb).sort(1).values
            want = torch.full((nqb, 8), -1)
            want[:, :pick.shape[1]] = torch.where(pick < nb, pick, -1).cpu()
            assert torch.equal(got[s, :nqb, h].long(), want), (s, h)
        at += n


@pytest.mark.parametrize("lens,H,HK,D,qb,block", [([200, 90], 16, 1, 128, 1, 64), ([300], 4, 2, 64, 16, 32), ([800], 4, 4, 64, 64, 64)])
def test_infinities_and_nan_stay_with_the_rows_that_read_them(lens, H, HK, D, qb, block):
    """Keys and values that are not finite, in blocks that some queries list and their neighbours do not: only rows that
    read such a key may notice.  Others equal the plain form over their own keys."""
    from cuspamm_b200 import block_sparse_attention

    g = torch.Generator().manual_seed(71)
    T = sum(lens)
    q, k, v, d_o = (tokens(g, T, n, D, BF) for n in (H, HK, HK, H))
    lists = random_lists(g, lens, lens, HK, block, qb, 2, True)
    k[70, 0, 3], k[110, 0, 5], v[75, 0, 1], v[131, 0] = torch.inf, torch.nan, -torch.inf, torch.nan
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    o = block_sparse_attention(*x, lists, cu_of(lens), max(lens), block=block, query_block=qb)
    (dq,) = torch.autograd.grad(o, x[:1], d_o)
    at, clean = 0, 0
    for s, n in enumerate(lens):
        r = slice(at, at + n)
        for h in range(H):
            hk = h // (H // HK)
            ok = plain.mask_of(lists[s].cpu(), n, n, 0, block, qb, True, hk).to(DEV)
            fine = torch.isfinite(k[r, hk]).all(1) & torch.isfinite(v[r, hk]).all(1)
            rows = ~(ok & ~fine[None]).any(1)                      # rows that read none of them
            clean += int(rows.sum())
            kk, vv = k[r, hk].nan_to_num(0, 0, 0), v[r, hk].nan_to_num(0, 0, 0)
            val, tol = plain.attend(q[r, h], kk, vv, ok, D ** -0.5, d_o[r, h])
            near(o[r, h][rows].detach(), val["o"][rows], tol["o"][rows], "o")
            near(dq[r, h][rows], val["dq"][rows], tol["dq"][rows], "dq")
        at += n
    assert clean > T                                              # most rows


def test_nan_of_a_later_token_of_a_short_chunk():
    """Four new tokens share a tile of rows; what the last one brings is seen by itself alone."""
    from cuspamm_b200 import PagedCache, block_sparse_attention

    g = torch.Generator().manual_seed(73)
    H, HK, D, page = 4, 2, 64, 16
    k, v, table, lengths = build_cache(g, [40], HK, D, HF, page)
    q, cu = tokens(g, 4, H, D, HF), cu_of([4])
    v[table[0, 39 // page].long(), :, 39 % page] = torch.nan
    k[table[0, 38 // page].long(), 1, 38 % page, 5] = torch.inf
    o = PagedCache(k, v).attend(q, cu, 4, table, lengths)
    for h in range(H):
        kk, vv = flat(k, table, 0, 40, h // 2).nan_to_num(0, 0, 0), flat(v, table, 0, 40, h // 2).nan_to_num(0, 0, 0)
        ok = plain.mask_of(None, 4, 40, 36, page, 1, True, h // 2).to(DEV)
        val, tol = plain.attend(q[:, h], kk, vv, ok, D ** -0.5)
        n = 3 if h < 2 else 2
        near(o[:n, h], val["o"][:n], tol["o"][:n], "o")
        assert bool(torch.isnan(o[3, h]).any())
    # the same in training: three tokens of one head
    q, k, v, d_o = (tokens(g, 3, 1, D, BF) for _ in range(4))
    v[2] = torch.inf
    x = q.clone().requires_grad_()
    lists = torch.zeros(1, 1, 1, 1, dtype=torch.int32, device=DEV)
    o = block_sparse_attention(x, k, v, lists, cu_of([3]), 3, block=16, query_block=16)
    (dq,) = torch.autograd.grad(o, x, d_o)
    val, tol = plain.attend(q[:2, 0], k[:2, 0], v[:2, 0], torch.ones(2, 2, dtype=torch.bool, device=DEV).tril(), D ** -0.5, d_o[:2, 0])
    near(o[:2, 0].detach(), val["o"], tol["o"], "o")
    near(dq[:2, 0], val["dq"], tol["dq"], "dq")


def test_offsets_beyond_four_gigabytes():
    """A cache whose last pages lie behind 2^32 bytes and 2^31 elements."""
    from cuspamm_b200 import PagedCache

    pages, HK, D, page = 36000, 8, 128, 64
    if torch.cuda.mem_get_info(0)[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    g = torch.Generator().manual_seed(81)
    k = torch.zeros(pages, HK, page, D, dtype=BF, device=DEV)
    v = torch.zeros_like(k)
    cache = PagedCache(k, v)
    held = [150, 70]
    table = torch.tensor([[35999, 0, 35998], [35997, 35000, 0]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor(held, dtype=torch.int32, device=DEV)
    nk, nv, q = tokens(g, 220, HK, D, BF), tokens(g, 220, HK, D, BF), tokens(g, 220, HK, D, BF)
    cache.append(nk, nv, cu_of(held), 150, table, lengths)
    for new in ([150, 70], [1, 1]):                               # the kernels of prompts and of single tokens
        qq = torch.cat([q[150 - new[0]:150], q[220 - new[1]:]])
        o = cache.attend(qq, cu_of(new), max(new), table, lengths)
        lists = cache.select(qq, cu_of(new), max(new), table, lengths, 3)
        assert sorted(set(lists.flatten().tolist())) == ([-1, 0, 1, 2] if new[0] > 1 else [-1, 0, 1, 2])
        listed = cache.attend(qq, cu_of(new), max(new), table, lengths, lists=lists)
        at, src = 0, 0
        for n, m in zip(held, new):
            for h in range(HK):
                ok = plain.mask_of(None, m, n, n - m, page, 1, True, h).to(DEV)
                val, tol = plain.attend(qq[at:at + m, h], nk[src:src + n, h], nv[src:src + n, h], ok, D ** -0.5)
                near(o[at:at + m, h], val["o"], tol["o"], "o")
                near(listed[at:at + m, h], val["o"], tol["o"], "listed")
            at, src = at + m, src + n
    cache.check()


@pytest.mark.parametrize("blocks", [300, 1025, 2048, 2049, 5000])
@pytest.mark.parametrize("ties", [False, True])
def test_select_of_new_tokens_over_many_pages(blocks, ties):
    """A few query blocks over every range of lengths that has a way of its own, with scores that mostly tie as well."""
    from cuspamm_b200 import PagedCache

    page, HK, G, D, new, n_select = 16, 2, 2, 64, [1, 3, 1], 40
    lens = [blocks * page, (blocks * page) // 3 + 1, 5]
    g = torch.Generator().manual_seed(blocks)
    k, v, table, lengths = build_cache(g, lens, HK, D, BF, page)
    cache = PagedCache(k, v)
    cache.key_sums.copy_(torch.randint(-1, 2, cache.key_sums.shape, generator=g) if ties else torch.randn(cache.key_sums.shape, generator=g))
    q = tokens(g, sum(new), HK * G, D, BF)
    if ties:
        q = torch.zeros_like(q)
        q[..., :2] = 1.0                     # scores of a few small whole numbers over 16
    got = cache.select(q, cu_of(new), max(new), table, lengths, n_select)
    cache.check()
    want, at = torch.full(got.shape, -1, dtype=torch.int32), 0
    for s, (n, m) in enumerate(zip(lens, new)):
        nb = -(-n // page)
        held = torch.tensor([min(page, n - b * page) for b in range(nb)])
        x = plain.lists_of(q[at:at + m].cpu(), cache.key_sums[table[s, :nb].long()].cpu(), held, n, n - m, page, 1, n_select, 1, 1, True)
        want[s, :x.shape[0]] = x
        at += m
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("lens,HK,G,n_select,block", [([2000, 1, 3000, 70], 2, 4, 16, 64), ([40, 900], 1, 16, 60, 16),
                                                      ([700], 1, 3, 0, 16), ([130, 260, 390], 2, 2, 0, 32)])
def test_ranges_joined_by_a_cluster(lens, HK, G, n_select, block):
    """Few rows whose keys are cut into a handful of ranges, some of them without keys, a NaN in one key that some rows read."""
    from cuspamm_b200 import PagedCache

    D, new = 128, [min(2, n) for n in lens]
    g = torch.Generator().manual_seed(sum(lens))
    k, v, table, lengths = build_cache(g, lens, HK, D, BF, block)
    last = int(table[0, (lens[0] - 1) // block])
    k[last, 0, (lens[0] - 1) % block, 3] = torch.nan               # the last token's key: only its own row sees it
    cache = PagedCache(k, v)
    q = tokens(g, sum(new), HK * G, D, BF)
    lists = None
    if n_select:
        lists = torch.full((len(lens), max(new), HK, n_select), -1, dtype=torch.int32)
        for s, n in enumerate(lens):
            nb = -(-n // block)
            for i in range(max(new)):
                for h in range(HK):
                    m = min(n_select, nb)
                    lists[s, i, h, :m] = torch.randperm(nb, generator=g)[:m].sort().values.int()
        lists[0, :, :, -1] = (lens[0] - 1) // block
        lists[0] = lists[0].sort(-1).values
        lists = lists.to(DEV)
    o, lse = cache.attend(q, cu_of(new), max(new), table, lengths, lists=lists, return_lse=True)
    cache.check()
    at = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        pages = table[s, :-(-n // block)].long()
        ks = k[pages].transpose(1, 2).reshape(-1, HK, D)[:n].double()
        vs = v[pages].transpose(1, 2).reshape(-1, HK, D)[:n].double()
        for i in range(m):
            for h in range(HK):
                ok = torch.arange(n, device=DEV) <= n - m + i
                if n_select:
                    ok &= torch.isin(torch.arange(n, device=DEV) // block, lists[s, i, h])
                z = (q[at + i, h * G:(h + 1) * G].double() @ ks[ok, h].T) * D ** -0.5
                want = torch.softmax(z, 1) @ vs[ok, h]
                got = o[at + i, h * G:(h + 1) * G].double()
                assert torch.equal(torch.isnan(got), torch.isnan(want))
                # p and o are rounded to bf16 (2^-8 each, relative to the sum of |p v| and to |o|); sums and exponentials in float
                bound = 2.0 ** -8 * (torch.softmax(z, 1) @ vs[ok, h].abs() + want.abs()) + 1e-4
                assert torch.isnan(want).any() or bool(((got - want).abs() <= bound).all()), (s, i, h)
                if not torch.isnan(z).any():
                    torch.testing.assert_close(lse[at + i, h * G:(h + 1) * G].double(), torch.logsumexp(z, 1), rtol=0, atol=1e-4)
        at += m
