"""Plain 64-bit forms of the attention operators for the tests, and how far the kernels may be from them.

The bounds count roundings.  u is half a step of the type (eps / 2).  The kernels round p (and ds) once to the type, a
relative error of u each, and the result once.  Scores are sums of D float products: their error is at most
D * 2^-24 * scale * sum |q||k|, which with D <= 128 and the inputs used here (sum |q||k| * scale below 16) is under
2^-13; it, and as much again for lse and the float sums, enters p as a relative error of SLACK = 2^-12.
"""
import torch

SLACK = 2.0 ** -12


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def kept(list_row, n_blocks):
    """The entries of a list that count: blocks of the sequence, each above every one before it."""
    out, top = [], -1
    for e in list_row:
        if 0 <= e < n_blocks and e > top:
            out.append(e)
            top = e
    return out


def mask_of(lists_s, nq, nk, pos0, block, query_block, causal, h):
    """[nq, nk] truth values of one sequence (lists_s [query blocks, kv_heads, n_select], or None: every block)."""
    key, pos = torch.arange(nk), pos0 + torch.arange(nq)
    ok = torch.ones(nq, nk, dtype=torch.bool)
    if lists_s is not None:
        ok[:] = False
        for i in range(nq):
            last = min((i // query_block + 1) * query_block, nq) - 1
            seen = min(max(pos0 + last + 1, 0), nk) if causal else nk
            for b in kept(lists_s[i // query_block, h].tolist(), -(-seen // block)):
                ok[i, b * block:(b + 1) * block] = True
    if causal:
        ok &= key[None, :] <= pos[:, None]
    return ok


def attend(q, k, v, ok, scale, d_o=None):
    """One head in 64 bits: q [nq, D], k, v [nk, D], ok [nq, nk].  Returns dicts of values and of bounds."""
    dt, u = q.dtype, half_step(q.dtype)
    q, k, v = q.double(), k.double(), v.double()
    z = (q @ k.T * scale).masked_fill(~ok, -torch.inf)
    lse = torch.logsumexp(z, 1) if z.shape[1] else torch.full((z.shape[0],), -torch.inf, dtype=torch.float64, device=q.device)
    p = torch.exp(z - torch.where(lse == -torch.inf, 0.0, lse)[:, None])
    o = p @ v
    weight = p @ v.abs()
    val, tol = dict(o=o, lse=lse), dict(o=(u + SLACK) * weight + u * o.abs() + 1e-7, lse=SLACK + 2.0 ** -22 * lse.abs().nan_to_num(0.0, posinf=0.0))
    if d_o is None:
        return val, tol
    g = d_o.double()
    dp, delta = g @ v.T, (g * o).sum(1, keepdim=True)
    ds = p * (dp - delta) * scale
    off_delta = (g.abs() * tol["o"]).sum(1, keepdim=True)              # delta comes from the rounded output
    off_ds = u * ds.abs() + p * scale * (off_delta + 2 * SLACK * (dp.abs() + delta.abs()))
    val.update(dq=ds @ k, dk=ds.T @ q, dv=p.T @ g)
    tol.update(dq=off_ds @ k.abs() + u * val["dq"].abs() + 1e-7, dk=off_ds.T @ q.abs() + u * val["dk"].abs() + 1e-7,
               dv=(u + SLACK) * (p.T @ g.abs()) + u * val["dv"].abs() + 1e-7)
    # half's smallest steps: what is rounded to below them is off by half of 2^-24, times what it meets
    if dt == torch.float16:
        tiny, n = 2.0 ** -25, ok.sum(1, keepdim=True).double()
        tol["o"] = tol["o"] + tiny * n * v.abs().max()
        tol["dq"] = tol["dq"] + tiny * (n * k.abs().max() + 1)
        m = ok.sum(0)[:, None].double()
        tol["dk"], tol["dv"] = tol["dk"] + tiny * (m * q.abs().max() + 1), tol["dv"] + tiny * (m * g.abs().max() + 1)
    return val, tol


def rotate(x, pos, inv_freq, interleaved):
    """x [tokens, heads, D] turned by pos, 64-bit angles, float cosines and sines, products and sums rounded to float."""
    r = inv_freq.numel()
    angle = pos.double()[:, None] * inv_freq.double()
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    y = x.float().clone()
    at = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if interleaved else (slice(0, r), slice(r, 2 * r))
    a, b = y[..., at[0]].clone(), y[..., at[1]].clone()
    y[..., at[0]], y[..., at[1]] = a * c - b * s, b * c + a * s
    return y.to(x.dtype)


def lists_of(q, key_sums, held, nk, pos0, block, query_block, n_select, n_first, n_local, causal):
    """The lists of one sequence: q [nq, H, D], key_sums [blocks, HK, D] float -> int32 [query blocks, HK, n_select]."""
    nq, HK = q.shape[0], key_sums.shape[1]
    nqb = -(-nq // query_block)
    out = torch.full((nqb, HK, n_select), -1, dtype=torch.int32)
    qs = q.double().view(nq, HK, q.shape[1] // HK, q.shape[2]).sum(2)
    for i in range(nqb):
        lo, hi = i * query_block, min((i + 1) * query_block, nq)
        first, last = pos0 + lo, pos0 + hi - 1
        seen = min(max(last + 1, 0), nk) if causal else nk
        n = -(-seen // block)
        forced = [b for b in range(n) if b < n_first or (n_local and first // block - n_local < b <= last // block)]
        for h in range(HK):
            score = (qs[lo:hi, h].sum(0) * key_sums[:n, h].double()).sum(1) / held[:n].double()
            rank = sorted((b for b in range(n) if b not in forced), key=lambda b: (-float(score[b]), b))
            take = sorted((forced + rank)[:n_select])
            out[i, h, :len(take)] = torch.tensor(take, dtype=torch.int32)
    return out
