"""Calls of the attention operators that the parity tests do not make: several host threads, other streams, sizes at the
borders of a launch, tensors with gradients, lengths beyond the table, kernels that only large problems reach."""
import threading

import pytest
import torch

import _attention_plain as plain
from test_gpu_attention import BF, DEV, HF, build_cache, cu_of, expect, flat, near, random_lists, tokens

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ shared memory of a launch

def calls_of_two_sizes(g):
    """For every kernel whose shared memory depends on the call: the same call large and small."""
    from cuspamm_b200 import PagedCache, block_sparse_attention, select_blocks

    def listed_attend(n_select):
        k, v, table, lengths = build_cache(g, [3000, 2000], 2, 128, BF, 16)
        q, lists = tokens(g, 2, 8, 128, BF), random_lists(g, [1, 1], [3000, 2000], 2, 16, 1, n_select, True)
        cache = PagedCache(k, v)
        return lambda: (cache.attend(q, cu_of([1, 1]), 1, table, lengths, lists=lists),)

    def select(n, block, query_block, heads, kv_heads):
        q, k = tokens(g, n, heads, 128, BF), tokens(g, n, kv_heads, 128, BF)
        return lambda: (select_blocks(q, k, cu_of([n]), n, 9, block=block, query_block=query_block, n_local=0),)

    def train(n, query_block, n_select, G):
        q, k, v, d_o = (tokens(g, n, h, 128, BF) for h in (2 * G, 2, 2, 2 * G))
        lists = random_lists(g, [n], [n], 2, 16, query_block, n_select, True)
        x = [t.requires_grad_() for t in (q, k, v)]

        def call():
            o = block_sparse_attention(*x, lists, cu_of([n]), n, block=16, query_block=query_block)
            return (o.detach(), *torch.autograd.grad(o, x, d_o))
        return call

    return [(listed_attend(150), listed_attend(8)),
            (select(16300, 16, 16, 2, 2), select(2100, 16, 16, 16, 16)),       # tiles of eight lists
            (select(4000, 16, 1, 2, 2), select(1600, 16, 1, 4, 4)),            # tiles of 32
            (select(130000, 16, 100, 1, 1), select(100000, 16, 80, 1, 1)),     # one list at a time
            (select(130000, 16, 50000, 1, 1), select(100000, 16, 50000, 1, 1)),
            (train(900, 16, 40, 4), train(200, 64, 4, 4)),
            (train(20, 16, 200, 1), train(20, 16, 2, 1))]                      # tiles of 16 rows


def test_two_host_threads_with_large_and_small_calls():
    """A kernel's limit of shared memory belongs to the process: one thread's small call must not undo another's large one."""
    g = torch.Generator().manual_seed(91)
    pairs = calls_of_two_sizes(g)
    want = [[call() for call in pair] for pair in pairs]
    torch.cuda.synchronize(DEV)
    trouble = []

    def repeat(which, times):
        try:
            for _ in range(times):
                for pair, results in zip(pairs, want):
                    for x, y in zip(pair[which](), results[which]):
                        assert torch.equal(x, y)
        except Exception as e:                                  # noqa: BLE001: handed to the test's own thread
            trouble.append(e)

    other = threading.Thread(target=repeat, args=(1, 1))        # a new thread sets the small limits; the large calls follow
    other.start()
    other.join()
    repeat(0, 1)
    both = [threading.Thread(target=repeat, args=(i % 2, 5)) for i in range(4)]
    for t in both:
        t.start()
    for t in both:
        t.join()
    assert not trouble, trouble

# D = 64: what the lists need beside the kernel's fixed shared memory comes to 48 KB and a little less
BORDERS = [(b, 64, 64, 8, 8) for b in (153, 154, 156, 157)] + [(b, 64, 1, 2, 2) for b in (54, 55, 56, 57)] + \
    [(b, 16, 64, 1, 1) for b in (6060, 6100, 6144, 6145)] + [(b, 16, 24576, 1, 1) for b in (6060, 6140, 6144, 6145)]


def check_selection(blocks, block, query_block, heads, kv_heads, D):
    from cuspamm_b200 import select_blocks

    n, n_select = blocks * block - 3, 9
    g = torch.Generator().manual_seed(blocks)
    q, k = tokens(g, n, heads, D, BF), tokens(g, n, kv_heads, D, BF)
    got = select_blocks(q, k, cu_of([n]), n, n_select, block=block, query_block=query_block, n_first=1, n_local=0)
    sums = torch.zeros(blocks, kv_heads, D, dtype=torch.float64, device=DEV).index_add_(0, torch.arange(n, device=DEV) // block, k.double())
    held = torch.full((blocks,), float(block), dtype=torch.float64, device=DEV)
    held[-1] = block - 3
    nqb = -(-n // query_block)
    qs = torch.zeros(nqb, kv_heads, D, dtype=torch.float64, device=DEV).index_add_(0, torch.arange(n, device=DEV) // query_block,
                                                                                             q.double().view(n, kv_heads, -1, D).sum(2))
    last = torch.clamp((torch.arange(nqb, device=DEV) + 1) * query_block, max=n) - 1
    seen = torch.arange(blocks, device=DEV)[None] * block <= last[:, None]
    for h in range(kv_heads):
        score = (qs[:, h] @ sums[:, h].float().double().T) / held
        score[:, 0] = torch.inf
        best = torch.where(seen, score, -torch.inf).topk(n_select, 1)
        want = torch.where(best.values > -torch.inf, best.indices, blocks).sort(1).values
        want = torch.where(want < blocks, want, -1)
        assert torch.equal(got[0, :, h].long(), want)


@pytest.mark.parametrize("blocks,block,query_block,heads,kv_heads", BORDERS)
def test_select_where_shared_memory_passes_48_kb(blocks, block, query_block, heads, kv_heads):
    check_selection(blocks, block, query_block, heads, kv_heads, 64)


# D = 128: tiles of 32 lists (4096 lists and more), of eight, one by one, spread
@pytest.mark.parametrize("blocks,block,query_block,heads,kv_heads", [(90, 64, 1, 2, 1), (255, 16, 1, 8, 2), (256, 32, 4, 4, 4), (1000, 16, 16, 4, 2),
                                                                     (1200, 16, 16, 1, 1), (700, 16, 5000, 2, 1)])
def test_select_with_heads_of_128(blocks, block, query_block, heads, kv_heads):
    check_selection(blocks, block, query_block, heads, kv_heads, 128)


# ------------------------------------------------------------------------------------------------ the largest numbers

@pytest.mark.parametrize("lens", [[2, 2, 1], [30, 20], [300, 200, 1]])
def test_one_list_for_the_whole_sequence(lens):
    """query_block of 2^31 - 1 is the same as one of the longest sequence, for every sequence and in both passes."""
    from cuspamm_b200 import PagedCache, block_sparse_attention, select_blocks

    g = torch.Generator().manual_seed(sum(lens))
    T, n, cu = sum(lens), max(lens), cu_of(lens)
    q, k, v, d_o = (tokens(g, T, h, 64, BF) for h in (4, 2, 2, 4))
    held = [x + 90 for x in lens]
    pages = build_cache(g, held, 2, 64, BF, 16)
    cache = PagedCache(*pages[:2])
    cache.key_sums.copy_(torch.randn(cache.key_sums.shape, generator=g))
    got = []
    for query_block in (n, 2 ** 31 - 1):
        lists = select_blocks(q, k, cu, n, 3, block=16, query_block=query_block, n_local=0)
        assert lists.shape == (len(lens), 1, 2, 3)
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        o = block_sparse_attention(*x, lists, cu, n, block=16, query_block=query_block)
        of_pages = cache.select(q, cu, n, *pages[2:], 3, query_block=query_block, n_local=0)
        got.append((lists, o.detach(), *torch.autograd.grad(o, x, d_o), of_pages,
                    cache.attend(q, cu, n, *pages[2:], lists=of_pages, query_block=query_block)))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    val, tol = expect(q, k, v, got[0][0], lens, 16, n, True, 64 ** -0.5, d_o)
    for name, x in zip(("o", "dq", "dk", "dv"), got[1][1:5]):
        near(x, val[name], tol[name], name)


# ------------------------------------------------------------------------------------------------ small numbers in half

@pytest.mark.parametrize("lens,H,HK,D,block,query_block,n_select", [([700, 90], 4, 2, 128, 64, 64, 8), ([300], 4, 4, 64, 16, 1, 6),
                                                                    ([20, 9], 1, 1, 128, 16, 5, 2), ([500], 16, 1, 64, 32, 1, 4)])
@pytest.mark.parametrize("size", [2.0 ** -13, 2.0 ** -7, 2.0 ** 11])
def test_half_gradients_keep_their_digits_whatever_the_size_of_the_output_gradient(lens, H, HK, D, block, query_block, n_select, size):
    """Output gradients of a small (or large) power of two times whole numbers: gradients are those of the whole numbers times
    that power, but for the rounding of the results themselves."""
    from cuspamm_b200 import block_sparse_attention

    g = torch.Generator().manual_seed(101)
    T, cu = sum(lens), cu_of(lens)
    q, k, v = (tokens(g, T, h, D, HF) for h in (H, HK, HK))
    whole = torch.randint(-8, 9, (T, H, D), generator=g).to(DEV)        # times 2^-3 to 2^-16 (half's last bit is 2^-24)
    lists = random_lists(g, lens, lens, HK, block, query_block, n_select, True)

    def gradients(d_o):
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        o = block_sparse_attention(*x, lists, cu, max(lens), block=block, query_block=query_block)
        return torch.autograd.grad(o, x, d_o)

    unit, small = gradients((whole * 2.0 ** -3).to(HF)), gradients((whole * 2.0 ** -3 * size).to(HF))
    u = plain.half_step(HF)
    for name, x, y in zip(("dq", "dk", "dv"), unit, small):
        # the roundings of the two results, and half's last bit (results near half's largest number are left out)
        want = x.double() * size
        near(torch.where(want.abs() < 6e4, y.double(), want), want, 2 * u * want.abs() + 2.0 ** -25 * (1 + size), name)


def test_half_gradients_of_long_flat_rows():
    """Rows over 4096 keys of nearly equal weight, output gradients of 1e-4: within roundings of the values, with nothing allowed
    for what half cannot hold but the last bit of the results."""
    from cuspamm_b200 import block_sparse_attention

    g = torch.Generator().manual_seed(103)
    n, D = 4096, 64
    q, k, v = (tokens(g, n, 1, D, HF) for _ in range(3))
    q *= 0.125
    d_o = (torch.randn(n, 1, D, generator=g) * 1e-4).to(HF).to(DEV)
    lists = torch.arange(64, dtype=torch.int32, device=DEV).expand(1, 64, 1, 64).contiguous()
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(block_sparse_attention(*x, lists, cu_of([n]), n, causal=False), x, d_o)
    ok = torch.ones(n, n, dtype=torch.bool, device=DEV)
    q, k, v, d_o = (t[:, 0].double() for t in (q, k, v, d_o))
    val, _ = plain.attend(q, k, v, ok, D ** -0.5, d_o)
    # half's roundings of p and ds (u each) and the float sums, as in _attention_plain.py
    u, p, dp, delta = plain.half_step(HF), torch.exp(q @ k.T * D ** -0.5 - val["lse"][:, None]), d_o @ v.T, (d_o * val["o"]).sum(1, keepdim=True)
    off_delta = (d_o.abs() * ((u + plain.SLACK) * (p @ v.abs()) + u * val["o"].abs())).sum(1, keepdim=True)
    off = u * (p * (dp - delta) * D ** -0.5).abs() + p * D ** -0.5 * (off_delta + 2 * plain.SLACK * (dp.abs() + delta.abs()))
    bound = dict(dq=off @ k.abs(), dk=off.T @ q.abs(), dv=(u + plain.SLACK) * (p.T @ d_o.abs()))
    for name, y in zip(("dq", "dk", "dv"), got):
        near(y[:, 0], val[name], bound[name] + u * val[name].abs() + 2.0 ** -25, name)


# ------------------------------------------------------------------------------------------------ gradients that do not exist

def test_a_backward_pass_through_the_cache_raises():
    """append and attend have no gradient: asking for it must not pass in silence."""
    from cuspamm_b200 import PagedCache

    g = torch.Generator().manual_seed(111)
    table, lengths, cu = torch.arange(2, dtype=torch.int32, device=DEV)[None], torch.tensor([20], dtype=torch.int32, device=DEV), cu_of([20])
    q, k, v = (tokens(g, 20, h, 64, BF) for h in (4, 2, 2))
    inv = torch.ones(32, device=DEV)

    def run(q, k, v, **kw):
        cache = PagedCache.empty(2, 2, 64, page_size=16, device=DEV)
        rq = cache.append(k, v, cu, 20, table, lengths, inv_freq=inv, q=q)
        return rq, cache.attend(q.detach() if kw.pop("cut", False) else rq, cu, 20, table, lengths, **kw)

    want = run(q, k, v)
    assert not want[0].requires_grad and not want[1].requires_grad
    with torch.no_grad():
        for x, y in zip(run(q.clone().requires_grad_(), k.clone().requires_grad_(), v), want):
            assert not x.requires_grad and torch.equal(x, y)
    w = q.clone().requires_grad_()
    got = run(w, k, v)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
        with pytest.raises(RuntimeError, match="no gradient"):
            x.float().sum().backward()
    assert w.grad is None
    for kw in (dict(k=k.clone().requires_grad_(), v=v), dict(k=k, v=v.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no gradient"):      # what was appended wanted one
            run(q, **kw, cut=True)[1].float().sum().backward()
    with pytest.raises(ValueError):
        run(w, k, v, out=torch.empty_like(q))
    with torch.no_grad():
        run(w, k, v, out=torch.empty_like(q))
    for x in run(w, k, v, return_lse=True)[1]:
        with pytest.raises(RuntimeError, match="no gradient"):
            x.float().sum().backward()


# ------------------------------------------------------------------------------------------------ reports

def test_check_waits_for_every_stream():
    """A bad page met on a stream that is not the current one, and that is busy when the report is asked for."""
    from cuspamm_b200 import PagedCache, SpammError

    g = torch.Generator().manual_seed(121)
    k, v, table, lengths = build_cache(g, [40], 1, 64, BF, 16)
    q, cu, cache = tokens(g, 1, 2, 64, BF), cu_of([1]), PagedCache(k, v)
    cache.attend(q, cu, 1, table, lengths)
    cache.check()
    table[0, 1] = -7
    torch.cuda.synchronize(DEV)
    side = torch.cuda.Stream(DEV)
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)                              # some 50 ms
        cache.attend(q, cu, 1, table, lengths)
    with pytest.raises(SpammError):
        cache.check()
    cache.check()


def test_calls_on_packed_tokens_report():
    """A sequence longer than the bound, and a wait given up (its code put in by hand), come out of check_attention once."""
    from cuspamm_b200 import SpammError, attention, block_sparse_attention, check_attention, select_blocks

    g = torch.Generator().manual_seed(131)
    q, k, v, d_o = (tokens(g, 50, h, 64, BF) for h in (2, 1, 1, 2))
    cu, lists = cu_of([30, 20]), torch.zeros(2, 1, 1, 1, dtype=torch.int32, device=DEV)
    check_attention()
    x = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(block_sparse_attention(*x, lists, cu, 30, block=16), x, d_o)
    select_blocks(q, k, cu, 30, 3, block=16, query_block=16)
    check_attention(DEV)
    o = block_sparse_attention(*x, lists, cu, 20, block=16)
    assert not bool(o[20:30].any()) and bool(o[30:].any())
    with pytest.raises(SpammError):
        check_attention()
    check_attention()
    cut = torch.autograd.grad(o, x, d_o)
    assert not any(bool(t[20:30].any()) for t in cut) and torch.equal(cut[0][30:], grads[0][30:])
    with pytest.raises(SpammError):
        check_attention()
    select_blocks(q, k, cu, 20, 3, block=16, query_block=16)
    with pytest.raises(SpammError):
        check_attention()
    check_attention()
    attention._STATUS[0].fill_(4)                                 # SPAMM_ERR_DEVICE_WAIT
    with pytest.raises(SpammError) as e:
        check_attention()
    assert e.value.status == 4
    check_attention()


# ------------------------------------------------------------------------------------------------ lists

@pytest.mark.parametrize("lens,H,HK,query_block", [([32], 1, 1, 32), ([33, 20], 1, 1, 40), ([17, 5], 4, 2, 17), ([300], 4, 2, 100)])
def test_unordered_lists_are_read_alike_by_every_tile_and_both_passes(lens, H, HK, query_block):
    """An entry counts when it is above every one before it, whether or not the rows of a tile reach it: all queries of a query
    block read the same blocks, up to their own position."""
    from cuspamm_b200 import block_sparse_attention

    g = torch.Generator().manual_seed(141)
    T, D, block = sum(lens), 64, 16
    q, k, v, d_o = (tokens(g, T, h, D, BF) for h in (H, HK, HK, H))
    nqb = -(-max(lens) // query_block)
    lists = torch.randint(-1, 1 + max(lens) // block, (len(lens), nqb, HK, 6), generator=g).int()
    lists[0, 0, :, :2] = torch.tensor([1, 0])
    lists = lists.to(DEV)
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    o, lse = block_sparse_attention(*x, lists, cu_of(lens), max(lens), block=block, query_block=query_block, return_lse=True)
    got = (o.detach(), lse, *torch.autograd.grad(o, x, d_o))
    val, tol = expect(q, k, v, lists, lens, block, query_block, True, D ** -0.5, d_o)
    for n, y in zip(("o", "lse", "dq", "dk", "dv"), got):
        near(y, val[n], tol[n], n)


# ------------------------------------------------------------------------------------------------ lengths beyond the table

@pytest.mark.parametrize("new", [1, 5, 40])
@pytest.mark.parametrize("beyond", [0, 1, 3, 100])
def test_tokens_beyond_the_table_are_left_out(new, beyond):
    """A sequence that outgrew its row of the table keeps what it holds: tokens without a page are not written (nor anything else
    instead), the others go to their own positions, queries see what there is up to theirs, and the report comes."""
    from cuspamm_b200 import PagedCache, SpammError

    g = torch.Generator().manual_seed(151)
    page, D, H, HK, room = 16, 64, 4, 2, 64
    k, v, table, _ = build_cache(g, [room, 10], HK, D, BF, page, nan_behind=False)
    cache = PagedCache(k.clone(), v.clone())
    cache.key_sums.fill_(3.0)
    held = [room + beyond, 10]
    lengths, cu = torch.tensor(held, dtype=torch.int32, device=DEV), cu_of([new, 2])
    q, nk, nv = (tokens(g, new + 2, h, D, BF) for h in (H, HK, HK))
    inv = (1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().to(DEV)
    rq = cache.append(nk, nv, cu, max(new, 2), table, lengths, inv_freq=inv, q=q)
    if beyond:
        with pytest.raises(SpammError):
            cache.check()
    want_k, want_v, want_s, want_q = k.clone(), v.clone(), torch.full_like(cache.key_sums, 3.0), torch.zeros_like(q)
    at = 0
    for s, n in enumerate((new, 2)):
        first = held[s] - n
        for i in range(n):
            p, pos = first + i, torch.tensor([first + i], device=DEV)
            if p >= room:
                continue
            want_q[at + i] = plain.rotate(q[at + i:at + i + 1], pos, inv, False)[0]
            want_k[table[s, p // page].long(), :, p % page] = plain.rotate(nk[at + i:at + i + 1], pos, inv, False)[0]
            want_v[table[s, p // page].long(), :, p % page] = nv[at + i]
        for b in range(first // page, -(-min(held[s], room) // page) if first < room else 0):
            want_s[table[s, b].long()] = want_k[table[s, b].long(), :, :min(page, held[s] - b * page)].double().sum(1).float()
        at += n
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v) and torch.equal(rq, want_q)
    assert torch.equal(cache.key_sums, want_s)
    o = cache.attend(q, cu, max(new, 2), table, lengths)
    lists = cache.select(q, cu, max(new, 2), table, lengths, 4, n_first=0, n_local=1)
    at = 0
    for s, n in enumerate((new, 2)):
        have, first = min(held[s], room), held[s] - n
        assert all((max(0, min(first + i + 1, have)) == 0) == (lists[s, i, 0, 0] < 0) for i in range(n))
        for h in range(H):
            ok = torch.arange(have, device=DEV)[None] <= first + torch.arange(n, device=DEV)[:, None]
            val, tol = plain.attend(q[at:at + n, h], flat(cache.k, table, s, have, h // 2), flat(cache.v, table, s, have, h // 2), ok, D ** -0.5)
            near(o[at:at + n, h], val["o"], tol["o"], "o")
        at += n


# ------------------------------------------------------------------------------------------------ values that are not finite

@pytest.mark.parametrize("what", ["q", "k", "qkv"])
def test_a_model_gone_to_nan_costs_no_more(what):
    """Rows whose own scores are NaN have NaN results and need no second look: a poisoned batch takes about its usual time."""
    from cuspamm_b200 import PagedCache, block_sparse_attention

    g = torch.Generator().manual_seed(161)
    n, H, HK, D = 2048, 8, 2, 128
    lists = random_lists(g, [n], [n], HK, 64, 64, 8, True)
    lists[:, :, :, 0] = 0                                           # (every query sees a key: none is empty)
    lists = lists.sort(-1).values.contiguous()
    k_pages, v_pages, table, lengths = build_cache(g, [4000], HK, D, BF, 64, nan_behind=False)
    cu, one = cu_of([n]), cu_of([1])

    def once(poison):
        q, k, v, d_o = (tokens(g, n, h, D, BF) for h in (H, HK, HK, H))
        cache = PagedCache(k_pages.clone(), v_pages.clone())
        if poison:
            for name, x in (("q", q), ("k", k), ("v", v), ("k", cache.k), ("v", cache.v)):
                if name in what:
                    x.fill_(torch.nan)
        x = [t.requires_grad_() for t in (q, k, v)]

        def calls():
            o = block_sparse_attention(*x, lists, cu, n)
            with torch.no_grad():
                return (o.detach(), *torch.autograd.grad(o, x[:1], d_o), cache.attend(q, cu, n, table, lengths),
                        cache.attend(q[:1], one, 1, table, lengths))
        return calls

    times = []
    for poison in (False, True):
        calls = once(poison)
        got = calls()
        if poison:
            assert all(bool(torch.isnan(y).all()) for y in got)
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        for _ in range(3):
            calls()
        end.record()
        torch.cuda.synchronize(DEV)
        times.append(start.elapsed_time(end))
    assert times[1] < 4 * times[0] + 1, times


# ------------------------------------------------------------------------------------------------ kernels of larger problems

@pytest.mark.parametrize("dtype,D,page", [(BF, 64, 16), (BF, 128, 64), (HF, 64, 128), (HF, 128, 32)])
@pytest.mark.parametrize("held,new", [([900, 130], [300, 130]), ([3100, 260, 1], [70, 260, 1])])
def test_chunks_in_pairs_of_tiles(dtype, D, page, held, new):
    """Unlisted chunks of many key heads: two tiles of 128 rows to a block of threads (148 pairs and more), an odd number of tiles, one
    range of keys or several, a page that is not there and a NaN in the last token's key and value."""
    from cuspamm_b200 import PagedCache, SpammError

    g = torch.Generator().manual_seed(171)
    HK, G = 8, 8 if len(new) == 2 else 6
    k, v, table, lengths = build_cache(g, held, HK, D, dtype, page)
    last = held[0] - 1
    k[table[0, last // page].long(), :, last % page, 1] = torch.nan
    v[table[0, last // page].long(), :, last % page, 2] = torch.nan
    gone = (held[0] - new[0]) // page // 2
    kept_table, kept = table.clone(), torch.ones(held[0], dtype=torch.bool, device=DEV)
    table[0, gone] = -3
    kept[gone * page:(gone + 1) * page] = False
    q, cu = tokens(g, sum(new), HK * G, D, dtype), cu_of(new)
    cache = PagedCache(k, v)
    o, lse = cache.attend(q, cu, max(new), table, lengths, return_lse=True)
    with pytest.raises(SpammError):
        cache.check()
    at = 0
    for s, (n, m) in enumerate(zip(held, new)):
        ok = plain.mask_of(None, m, n, n - m, page, 1, True, 0).to(DEV)
        rows = m
        if s == 0:
            ok &= kept[None]
            rows = m - 1                                            # the last query reads the NaN
            assert bool(torch.isnan(o[at + rows]).all()) and bool(torch.isnan(lse[at + rows]).all())
        for h in range(HK * G):
            kk, vv = (flat(x, kept_table, s, n, h // G).nan_to_num(0.0) for x in (k, v))
            val, tol = plain.attend(q[at:at + rows, h], kk, vv, ok[:rows], D ** -0.5)
            near(o[at:at + rows, h], val["o"], tol["o"], f"o {s} {h}")
            near(lse[at:at + rows, h], val["lse"], tol["lse"], f"lse {s} {h}")
        at += m


@pytest.mark.parametrize("lens,H,HK,D,dtype,block,query_block,n_select,causal", [
    ([1100], 16, 1, 128, BF, 64, 1, 3, True), ([1100], 16, 1, 64, HF, 128, 1, 2, True), ([1300, 40], 16, 1, 128, HF, 128, 1, 2, False),
    ([700], 16, 1, 64, BF, 16, 1, 4, True), ([1200, 3], 32, 2, 128, BF, 32, 1, 3, True), ([700], 64, 2, 64, HF, 64, 2, 2, True)])
def test_blocks_that_very_many_queries_list(lens, H, HK, D, dtype, block, query_block, n_select, causal):
    """Every query lists block 0: its gradients are sums of several work items, joined."""
    from cuspamm_b200 import block_sparse_attention

    g = torch.Generator().manual_seed(181)
    T = sum(lens)
    q, k, v, d_o = (tokens(g, T, h, D, dtype) for h in (H, HK, HK, H))
    lists = random_lists(g, lens, lens, HK, block, query_block, n_select, causal)
    lists[..., 0] = 0
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    o = block_sparse_attention(*x, lists, cu_of(lens), max(lens), block=block, query_block=query_block, causal=causal)
    got = (o.detach(), *torch.autograd.grad(o, x, d_o))
    val, tol = expect(q, k, v, lists, lens, block, query_block, causal, D ** -0.5, d_o)
    for n, y in zip(("o", "dq", "dk", "dv"), got):
        near(y, val[n], tol[n], n)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype,lens,H,HK,query_block,causal", [(BF, [300, 77], 4, 2, 32, True), (HF, [290], 3, 1, 128, False)])
def test_every_block_and_head_size(dtype, D, block, lens, H, HK, query_block, causal):
    from cuspamm_b200 import block_sparse_attention

    g = torch.Generator().manual_seed(191 + D + block)
    T = sum(lens)
    q, k, v, d_o = (tokens(g, T, h, D, dtype) for h in (H, HK, HK, H))
    lists = random_lists(g, lens, lens, HK, block, query_block, 4, causal)
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    o = block_sparse_attention(*x, lists, cu_of(lens), max(lens), block=block, query_block=query_block, causal=causal)
    got = (o.detach(), *torch.autograd.grad(o, x, d_o))
    val, tol = expect(q, k, v, lists, lens, block, query_block, causal, D ** -0.5, d_o)
    for n, y in zip(("o", "dq", "dk", "dv"), got):
        near(y, val[n], tol[n], n)


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, HF)])
def test_lists_over_more_blocks_than_one_union_holds(D, dtype):
    """Ten thousand blocks of 16 keys: the tiles' unions in two ranges, dq in tiles of 16 rows. Sampled queries and blocks against
    the plain form over the listed keys."""
    from cuspamm_b200 import block_sparse_attention

    g = torch.Generator().manual_seed(201)
    n, block, query_block, n_select, G = 160005, 16, 48, 5, 2
    q, k, v, d_o = (tokens(g, n, h, D, dtype) for h in (G, 1, 1, G))
    nqb, nkb = -(-n // query_block), -(-n // block)
    own = (torch.arange(nqb) * query_block + query_block - 1).clamp(max=n - 1) // block
    lists = (torch.rand(nqb, n_select, generator=g) * own[:, None]).long()
    lists[:, 0], lists[:, -1] = torch.randint(0, 3, (nqb,), generator=g), own
    lists = lists.sort(1).values.int()
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    o = block_sparse_attention(*x, lists[None, :, None].contiguous().to(DEV), cu_of([n]), n, block=block, query_block=query_block)
    got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, x, d_o))))
    rows_of = lambda i: torch.arange(i * query_block, min((i + 1) * query_block, n), device=DEV)  # noqa: E731

    def of_query_block(i, h):
        keys = torch.cat([torch.arange(b * block, min((b + 1) * block, n), device=DEV) for b in sorted(set(lists[i].tolist()))])
        rows = rows_of(i)
        return rows, keys, *plain.attend(q[rows, h], k[keys, 0], v[keys, 0], keys[None] <= rows[:, None], D ** -0.5, d_o[rows, h])

    for i in [0, 1, 2000, nqb // 2, nqb - 2, nqb - 1]:
        for h in range(G):
            rows, _, val, tol = of_query_block(i, h)
            for name in ("o", "dq"):
                near(got[name][rows, h], val[name], tol[name], f"{name} {i}")
    for b in [3000, nkb // 2, nkb - 1]:
        at = torch.arange(b * block, min((b + 1) * block, n), device=DEV)
        val, tol = ({name: torch.zeros(len(at), D, dtype=torch.float64, device=DEV) for name in ("dk", "dv")} for _ in range(2))
        for i in (lists == b).any(1).nonzero()[:, 0].tolist():
            for h in range(G):
                _, keys, x, t = of_query_block(i, h)
                here = (keys // block == b).nonzero()[:, 0]
                for name in ("dk", "dv"):
                    val[name] += x[name][here]
                    tol[name] += t[name][here]
        for name in ("dk", "dv"):
            near(got[name][at, 0], val[name], tol[name], f"{name} {b}")


def test_the_exponential_by_polynomial():
    """lse of rows with two keys that count, scores 0 and x: log(1 + e^x), the second key in every place of a tile."""
    from cuspamm_b200 import PagedCache

    g = torch.Generator().manual_seed(211)
    held, new, D = 256, 64, 64
    table, lengths, cu = torch.arange(4, dtype=torch.int32, device=DEV)[None], torch.tensor([held], dtype=torch.int32, device=DEV), cu_of([new])
    k = torch.zeros(4, 1, 64, D, dtype=BF, device=DEV)
    q = torch.zeros(new, 1, D, dtype=BF, device=DEV)
    q[:, 0, 0] = 1.0
    for place in range(1, 128):
        k.zero_()
        k[..., 0] = -1000.0                                         # e^-1000: nothing
        k[0, 0, 0] = 0.0
        k[place // 64, 0, place % 64, 0], k[place // 64, 0, place % 64, 1] = 0.0, 1.0
        q[:, 0, 1] = (-15 * torch.rand(new, generator=g)).to(BF)
        _, lse = PagedCache(k, k).attend(q, cu, new, table, lengths, scale=1.0, return_lse=True)
        x = q[:, 0, 1].double()
        e = torch.exp(x)
        # 2.7e-6 of the polynomial, the exponent's rounding (two of 2^-24 of a number up to 22, times ln 2), two steps of a sum
        # between 1 and 2, its logarithm and the product with ln 2
        bound = e / (1 + e) * (2.7e-6 + 2.0 ** -23 * x.abs() + 2.0 ** -23) + 4 * 2.0 ** -24
        off = (lse[:, 0].double() - torch.log1p(e)).abs() - bound
        assert float(off.max()) <= 0, (place, float(off.max()))


def test_half_gradients_with_very_large_scores():
    """Scores of 10^7, where a float's last bit is one: the largest takes all the weight, and nothing overflows."""
    from cuspamm_b200 import block_sparse_attention

    g = torch.Generator().manual_seed(221)
    n, D = 64, 64
    q, k, v, d_o = (tokens(g, n, 1, D, HF) for _ in range(4))
    q, k = q * 600, k * 600
    lists = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV).expand(1, 4, 1, 4).contiguous()
    x = [t.detach().requires_grad_() for t in (q, k, v)]
    o = block_sparse_attention(*x, lists, cu_of([n]), n, block=16, query_block=16, scale=1.0)
    got = torch.autograd.grad(o, x, d_o)
    z = (q[:, 0].double() @ k[:, 0].double().T).masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), -torch.inf)
    best = z.argmax(1)
    two = z.topk(2, 1).values
    assert float((two[1:, 0] - two[1:, 1]).min()) > 2 ** 5 and float(z.max()) > 1e7
    near(o[:, 0].detach(), v[best, 0], 2.0 ** -10 * v[best, 0].double().abs(), "o")
    assert all(bool(torch.isfinite(y).all()) for y in got)
    # p is one but for its exponent's roundings: below 2^24 in powers of two, each is off by one at the most, and there are four
    # (the running maximum, lse in units of e and back, the difference): p is within 2^4 of one
    want = torch.zeros(n, D, dtype=torch.float64, device=DEV).index_add_(0, best, d_o[:, 0].double().abs())
    assert float(z.max()) * 1.4427 < 2 ** 24 + 2 ** 23
    assert float((got[2][:, 0].double().abs() - 16 * want).max()) <= 2.0 ** -10


@pytest.mark.parametrize("what", ["v", "k"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_an_infinity_that_every_row_reads_costs_no_more(what, dtype):
    """The first token's value (or key) is infinite in one column, and every query reads it: its column of o (of dq) is not finite,
    the others are as they should be, and nothing takes much longer."""
    from cuspamm_b200 import PagedCache, block_sparse_attention

    g = torch.Generator().manual_seed(231)
    n, H, HK, D, COL = 2048, 8, 2, 128, 5
    lists = random_lists(g, [n], [n], HK, 64, 64, 8, True)
    lists[..., 0] = 0
    q, k, v, d_o = (tokens(g, n, h, D, dtype) for h in (H, HK, HK, H))
    pages_k, pages_v, table, lengths = build_cache(g, [4000], HK, D, dtype, 64, nan_behind=False)
    cu, one = cu_of([n]), cu_of([1])
    finite = [t.clone() for t in (k, v, pages_k, pages_v)]
    first = table[0, 0].long()

    def times():
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        cache = PagedCache(pages_k, pages_v)

        def calls():
            o = block_sparse_attention(*x, lists, cu, n)
            with torch.no_grad():
                return (o.detach(), *torch.autograd.grad(o, x[:1], d_o), cache.attend(q, cu, n, table, lengths),
                        cache.attend(q[-1:], one, 1, table, lengths))
        got = calls()
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        for _ in range(3):
            calls()
        end.record()
        torch.cuda.synchronize(DEV)
        return got, start.elapsed_time(end)

    usual = times()[1]
    for x in ((v[0], pages_v[first, :, 0]) if what == "v" else (k[0], pages_k[first, :, 0])):
        x[..., COL] = torch.inf
    got, took = times()
    assert took < 4 * usual + 1, (took, usual)
    rest = [c for c in range(D) if c != COL]
    fk, fv, pk, pv = finite
    for h in range(H):
        hk = h // (H // HK)
        ok = plain.mask_of(lists[0].cpu()[None][0], n, n, 0, 64, 64, True, hk).to(DEV)
        over_pages = torch.arange(4000, device=DEV)[None] <= (4000 - n + torch.arange(n, device=DEV))[:, None]
        rows = slice(0, n)
        if what == "k":
            # a score of minus infinity: the key has no weight (plus infinity: all is NaN)
            rows = (q[:, h, COL] < 0) & (torch.arange(n, device=DEV) > 0)
            lost = q[:, h, COL] >= 0
            assert all(bool(torch.isnan(y[:, h][lost]).all()) for y in got[:3])
            ok[:, 0], over_pages[:, 0] = False, False
        val, tol = plain.attend(q[rows, h], fk[:, hk], fv[:, hk], ok[rows], D ** -0.5, d_o[rows, h])
        if what == "v":
            assert bool(got[0][:, h, COL].isinf().all()) and not bool(got[1][:, h].isfinite().any())
            near(got[0][:, h][:, rest], val["o"][:, rest], tol["o"][:, rest], "o")
        else:
            near(got[0][rows, h], val["o"], tol["o"], "o")
            near(got[1][rows, h][:, rest], val["dq"][:, rest], tol["dq"][:, rest], "dq")
            assert not bool(got[1][rows, h, COL].isfinite().any())
        val, tol = plain.attend(q[rows, h], flat(pk, table, 0, 4000, hk), flat(pv, table, 0, 4000, hk), over_pages[rows], D ** -0.5)
        columns = rest if what == "v" else list(range(D))
        near(got[2][rows, h][:, columns], val["o"][:, columns], tol["o"][:, columns], "over pages")
        if what == "v" or bool(q[-1, h, COL] < 0):
            near(got[3][0, h, columns], val["o"][-1, columns], tol["o"][-1, columns], "one token")
            assert what == "k" or bool(got[3][0, h, COL].isinf())


# ------------------------------------------------------------------------------------------------ layouts

def test_rows_before_between_and_behind_the_sequences():
    """cu_seqlens that begins behind row 0 and ends before the last: rows of no sequence are zero, in results and gradients, and what
    stands in them (NaN) changes nothing."""
    from cuspamm_b200 import block_sparse_attention, select_blocks

    g = torch.Generator().manual_seed(241)
    lens, lead, tail, H, HK, D = [60, 0, 75], 5, 9, 4, 2, 64
    T = lead + sum(lens) + tail
    for dtype in (BF, HF):
        q, k, v, d_o = (tokens(g, T, h, D, dtype) for h in (H, HK, HK, H))
        inner = slice(lead, T - tail)
        lists = random_lists(g, lens, lens, HK, 16, 16, 3, True)

        def run(q, k, v, d_o, cu):
            x = [t.detach().requires_grad_() for t in (q, k, v)]
            o = block_sparse_attention(*x, lists, cu, 75, block=16, query_block=16)
            return (o.detach(), *torch.autograd.grad(o, x, d_o)), select_blocks(q, k, cu, 75, 4, block=16, query_block=16)

        want, picked = run(*(t[inner].clone() for t in (q, k, v, d_o)), cu_of(lens))
        for t in (q, k, v, d_o):
            t[:lead], t[T - tail:] = torch.nan, torch.inf
        got, again = run(q, k, v, d_o, cu_of(lens) + lead)
        assert torch.equal(picked, again)
        for a, b in zip(want, got):
            assert torch.equal(a, b[inner]) and not bool(b[:lead].any()) and not bool(b[T - tail:].any())


@pytest.mark.parametrize("new,n_select", [([1, 1], 0), ([1, 1], 5), ([130, 70], 0), ([130, 70], 5)])
def test_results_into_strided_rows_and_tables_cut_from_wider_ones(new, n_select):
    """out= with gaps between rows and heads, out= over q itself, a page table whose rows are part of a wider one."""
    from cuspamm_b200 import PagedCache

    g = torch.Generator().manual_seed(251)
    H, HK, D, page = 8, 2, 128, 16
    k, v, table, lengths = build_cache(g, [700, 333], HK, D, BF, page)
    wide = torch.full((2, table.shape[1] + 7), 2 ** 30, dtype=torch.int32, device=DEV)
    wide[:, 3:3 + table.shape[1]] = table
    q, cu, cache = tokens(g, sum(new), H, D, BF), cu_of(new), PagedCache(k, v)
    lists = random_lists(g, new, [700, 333], HK, page, 1, n_select, True) if n_select else None
    want = cache.attend(q, cu, max(new), table, lengths, lists=lists)
    assert torch.equal(cache.attend(q, cu, max(new), wide[:, 3:3 + table.shape[1]], lengths, lists=lists), want)
    room = torch.full((sum(new), 2 * H, D + 8), 7.0, dtype=BF, device=DEV)
    out = room[:, ::2, :D]
    assert cache.attend(q, cu, max(new), table, lengths, lists=lists, out=out) is out
    assert torch.equal(out, want) and bool((room[:, 1::2] == 7.0).all()) and bool((room[..., D:] == 7.0).all())
    same = q.clone()
    assert torch.equal(cache.attend(same, cu, max(new), table, lengths, lists=lists, out=same), want)
    cache.check()
