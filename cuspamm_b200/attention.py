"""Attention over selected blocks: the engine's scheme (a cheap score for every block, lists of the blocks worth
multiplying, products of the listed blocks only) for queries, keys and values on the GPU.

    lists = select_blocks(q, k, cu_seqlens, max_seqlen, n_select)
    o = block_sparse_attention(q, k, v, lists, cu_seqlens, max_seqlen)        # differentiable in q, k and v
    check_attention()                                                         # now and then: what the kernels reported

and, for serving, over a paged cache whose pages are the blocks:

    cache = PagedCache.empty(n_pages, kv_heads, head_dim)
    q = cache.append(k, v, cu_seqlens, max_new, page_table, lengths, inv_freq=inv_freq, q=q)
    lists = cache.select(q, cu_seqlens, max_new, page_table, lengths, n_select)
    o = cache.attend(q, cu_seqlens, max_new, page_table, lengths, lists=lists)   # or lists=None: all pages

Tensors are torch tensors on one GPU, bf16 or half; work is queued on torch's current stream of that GPU, memory comes
from torch's allocator, nothing is read back, and every call may be captured into a CUDA graph.  Tokens of all sequences
lie one behind the other: q is [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim], sequence s the rows
cu_seqlens[s] .. cu_seqlens[s+1] - 1 (int32 on the GPU).  Views are fine as long as the last dimension is contiguous and
rows begin on 16-byte boundaries.  There is no counterpart in the reference.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from ._lib import SpammAttn, SpammError, check

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_BLOCKS = (16, 32, 64, 128)


def _rows(name: str, x: torch.Tensor, heads: Optional[int] = None, like: Optional[torch.Tensor] = None):
    """Checks a tensor of rows; its token and head stride (those of a dimension of one element are never used: 0)."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if x.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name} must be bfloat16 or float16, got {x.dtype}")
    n_tokens, n_heads, dim = x.shape
    if dim != 64 and dim != 128:
        raise ValueError(f"{name}: head_dim must be 64 or 128, got {dim}")
    if heads is not None and n_heads != heads:
        raise ValueError(f"{name} must have {heads} heads, got {n_heads}")
    if like is not None:
        tokens, _, like_dim = like.shape
        if n_tokens != tokens or dim != like_dim or x.dtype != like.dtype or x.device != like.device:
            raise ValueError(f"{name} must match in tokens, head_dim, dtype and device: {tuple(x.shape)} {x.dtype} {x.device} "
                             f"against {tuple(like.shape)} {like.dtype} {like.device}")
    token, head, last = x.stride()
    if last != 1 and x.numel():
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return token if n_tokens > 1 else 0, head if n_heads > 1 else 0


def _ints(name: str, x: torch.Tensor, shape, device) -> torch.Tensor:
    if not isinstance(x, torch.Tensor) or x.dtype != torch.int32:
        raise ValueError(f"{name} must be an int32 tensor")
    if x.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} must be on {device}, is on {x.device}")
    if not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return x


def _host_int(name: str, x, least: int = 0) -> int:
    if type(x) is int and least <= x < 2 ** 31:
        return x
    if isinstance(x, torch.Tensor):
        raise TypeError(f"{name} is a host-side number, not a tensor")
    v = int(x)
    if v != x or not least <= v < 2 ** 31:
        raise ValueError(f"{name} must be a whole number of at least {least}, got {x}")
    return v


def _on_gpu(x: torch.Tensor) -> None:
    if not x.is_cuda:
        raise ValueError(f"tensors must be on a GPU, got {x.device}")


def _like(x: torch.Tensor) -> torch.Tensor:
    """A new tensor of x's shape without gaps."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _problem(q: torch.Tensor, q_strides, kv_heads: int, cu_seqlens: torch.Tensor, max_q: int, block: int, query_block: int,
             causal: bool) -> SpammAttn:
    tokens, heads, dim = q.shape
    if block not in _BLOCKS:
        raise ValueError(f"block must be one of {_BLOCKS}, got {block}")
    if kv_heads < 1 or heads % kv_heads or not 1 <= heads // kv_heads <= 128:
        raise ValueError(f"{heads} query heads for {kv_heads} key heads: must be a multiple, 1 to 128 times")
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be a tensor [batch + 1]")
    _ints("cu_seqlens", cu_seqlens, cu_seqlens.shape, q.device)
    a = SpammAttn()                          # all zeros
    a.dtype = _DTYPES[q.dtype]
    a.batch = cu_seqlens.shape[0] - 1
    a.heads = heads
    a.kv_heads = kv_heads
    a.dim = dim
    a.block = block
    a.query_block = query_block
    a.causal = 1 if causal else 0
    a.max_q = max_q
    a.tokens = tokens
    a.zero_tail = 1
    a.scale = 1.0
    a.d_cu = cu_seqlens.data_ptr()
    a.d_q = q.data_ptr()
    a.q_token, a.q_head = q_strides
    return a


_STATUS = {}           # device index -> the word in which the calls on packed tokens leave what went wrong


def _packed_status(device) -> Optional[int]:
    status = _STATUS.get(device.index)
    if status is None:
        if torch.cuda.is_current_stream_capturing():
            return None              # a capture before any call outside one: its memory would belong to the graph
        stream = torch.cuda.Stream(device)
        with torch.cuda.stream(stream):
            status = torch.zeros(1, dtype=torch.int32, device=device)
        stream.synchronize()
        status = _STATUS.setdefault(device.index, status)
    return status.data_ptr()


def check_attention(device=None) -> None:
    """Waits for the GPU (for the work of all streams) and raises SpammError when a `select_blocks` or
    `block_sparse_attention` call on it, or a backward pass of one, met a sequence longer than `max_seqlen`, or gave up a wait
    inside a kernel (its result is then NaN), since the last report.  (PagedCache.check reports for the cache's calls.)"""
    index = torch.device("cuda" if device is None else device).index
    status = _STATUS.get(torch.cuda.current_device() if index is None else index)
    if status is not None:
        _report(status, "attention")


def _set_keys(a: SpammAttn, k: torch.Tensor, k_strides, v: Optional[torch.Tensor] = None, v_strides=None) -> None:
    a.d_k = k.data_ptr()
    a.k_token, a.k_head = k_strides
    if v is not None:
        a.d_v = v.data_ptr()
        a.v_token, a.v_head = v_strides


def _set_out(a: SpammAttn, o: torch.Tensor) -> None:
    """o without gaps."""
    a.d_o = o.data_ptr()
    a.o_token = a.heads * a.dim
    a.o_head = a.dim


def _set_lists(a: SpammAttn, lists: torch.Tensor, device) -> None:
    if not isinstance(lists, torch.Tensor) or lists.dim() != 4:
        raise ValueError("lists must be a tensor [batch, query blocks, kv_heads, n_select]")
    if not 1 <= lists.shape[3] <= 1024:
        raise ValueError(f"lists of {lists.shape[3]} entries: 1 to 1024 are possible")
    _ints("lists", lists, (a.batch, -(-a.max_q // a.query_block), a.kv_heads, lists.shape[3]), device)
    a.n_select = lists.shape[3]
    a.d_lists = lists.data_ptr()


def _scratch(nbytes: int, device):
    t = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    return t, (t.data_ptr() if nbytes else None)


def _scale(scale, head_dim: int) -> float:
    s = head_dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < s < 3e38:
        raise ValueError(f"scale must be a positive number, got {scale}")
    return s


def _stream(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


class _Same:
    """Stands for torch.cuda.device where the tensors' device is the current one already."""

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_SAME = _Same()


def _device(device):
    return _SAME if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _select(a: SpammAttn, q: torch.Tensor, key_sums: Optional[torch.Tensor], n_select, n_first, n_local) -> torch.Tensor:
    lib = _lib.load()
    forced = n_first + (n_local + (a.query_block + a.block - 2) // a.block if n_local else 0)
    if not 1 <= n_select <= 1024 or n_select < forced:
        raise ValueError(f"n_select must be 1 to 1024 and hold the {forced} first and local blocks, got {n_select}")
    a.n_select = n_select
    _on_gpu(q)
    with _device(q.device):
        if not a.n_pages:
            a.d_status = _packed_status(q.device)
        lists = torch.empty((a.batch, -(-a.max_q // a.query_block), a.kv_heads, n_select), dtype=torch.int32, device=q.device)
        n = lib.spamm_attn_select_scratch_bytes(C.byref(a))
        scratch, ptr = _scratch(n, q.device)
        check(lib.spamm_attn_select_dev(C.byref(a), key_sums.data_ptr() if key_sums is not None else None, n_first, n_local,
                                        lists.data_ptr(), ptr, n, _stream(q.device)), "spamm_attn_select_dev")
    return lists


def _forward(a: SpammAttn, device) -> None:
    lib = _lib.load()
    n = lib.spamm_attn_forward_scratch_bytes(C.byref(a))
    scratch, ptr = _scratch(n, device)
    check(lib.spamm_attn_forward_dev(C.byref(a), ptr, n, _stream(device)), "spamm_attn_forward_dev")


def select_blocks(q: torch.Tensor, k: torch.Tensor, cu_seqlens: torch.Tensor, max_seqlen: int, n_select: int, *,
                  block: int = 64, query_block: int = 64, n_first: int = 1, n_local: int = 1,
                  causal: bool = True) -> torch.Tensor:
    """Lists of the `n_select` blocks of `block` keys with the largest scores, one list for every `query_block`
    consecutive queries (1: every query its own) and key head: int32 [batch, ceil(max_seqlen / query_block), kv_heads,
    n_select], ascending, -1 behind.  The score of a block is the sum of the queries (over the query block and the heads
    of the key head) times the block's mean key; it is taken in double, ties go to the lower block.  The first `n_first`
    blocks and those from `n_local` - 1 before the first query's to the last query's own are always taken.  No sequence
    may be longer than `max_seqlen` (`check_attention` reports it; what is beyond is left out).  The choice is not
    differentiable."""
    q_strides = _rows("q", q)
    k_strides = _rows("k", k, like=q)
    a = _problem(q, q_strides, k.shape[1], cu_seqlens, _host_int("max_seqlen", max_seqlen), _host_int("block", block),
                 _host_int("query_block", query_block, 1), causal)
    _set_keys(a, k, k_strides)
    return _select(a, q, None, _host_int("n_select", n_select, 1), _host_int("n_first", n_first), _host_int("n_local", n_local))


def _own_strides(x: torch.Tensor):
    (tokens, heads, _), (token, head, _) = x.shape, x.stride()
    return token if tokens > 1 else 0, head if heads > 1 else 0


class _BlockSparseAttention(torch.autograd.Function):
    """`a` describes q, k, v, the lists and cu_seqlens, checked."""

    @staticmethod
    def forward(ctx, q, k, v, lists, cu_seqlens, a, want_lse):
        device = q.device
        with _device(device):
            a.d_status = _packed_status(device)
            o = _like(q)
            lse = torch.empty((a.tokens, a.heads), dtype=torch.float32, device=device)
            _set_out(a, o)
            a.d_lse = lse.data_ptr()
            # what the rounding of o left, for the backward's do.o: only where there will be one
            low = _like(q) if any(ctx.needs_input_grad[:3]) else None
            a.d_o_low = low.data_ptr() if low is not None else None
            if not a.batch or not a.max_q:
                o.zero_()
                lse.fill_(float("-inf"))
            _forward(a, device)
        if low is not None:
            ctx.save_for_backward(q, k, v, lists, cu_seqlens, o, low, lse)
            ctx.problem = a
        if not want_lse:
            return o
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, *_):
        q, k, v, lists, cu_seqlens, o, low, lse = ctx.saved_tensors
        # the sizes are the forward's; the tensors may lie elsewhere by now (hooks on saved tensors)
        a = SpammAttn.from_buffer_copy(ctx.problem)
        a.d_q, a.d_o = q.data_ptr(), o.data_ptr()
        a.q_token, a.q_head = _own_strides(q)
        a.o_token, a.o_head = _own_strides(o)
        _set_keys(a, k, _own_strides(k), v, _own_strides(v))
        a.d_lists, a.d_cu = lists.data_ptr(), cu_seqlens.data_ptr()
        a.d_lse, a.d_o_low = lse.data_ptr(), low.data_ptr()
        # an expanded or oddly laid out gradient (the sum's, for one) is brought into rows first
        do_token, do_head = _own_strides(d_o)
        if (d_o.stride(2) != 1 or d_o.data_ptr() % 16 or do_token % 8 or do_head % 8) and d_o.numel():
            d_o = d_o.contiguous()
            do_token, do_head = _own_strides(d_o)
        lib = _lib.load()
        device = q.device
        with _device(device):
            dq, dk, dv = _like(q), _like(k), _like(k)
            n = lib.spamm_attn_backward_scratch_bytes(C.byref(a))
            scratch, ptr = _scratch(n, device)
            check(lib.spamm_attn_backward_dev(C.byref(a), d_o.data_ptr(), do_token, do_head, dq.data_ptr(), dk.data_ptr(),
                                              dv.data_ptr(), ptr, n, _stream(device)), "spamm_attn_backward_dev")
        return dq, dk, dv, None, None, None, None


def block_sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lists: torch.Tensor, cu_seqlens: torch.Tensor,
                           max_seqlen: int, *, block: int = 64, query_block: int = 64, causal: bool = True,
                           scale: Optional[float] = None, return_lse: bool = False):
    """Attention of every query over the keys of the blocks on its query block's list (`lists` as `select_blocks` gives
    them; an entry that is no block which some query of the query block may see, or not above every such entry before it,
    is skipped), with `causal` over those up to its own position.  `scale` multiplies q.k (default head_dim ** -0.5).  A
    query that sees no key gets zeros.  Returns o [tokens, heads, head_dim], with `return_lse` also the log of the sum of
    exp(scale * q.k) per query and head (float, not differentiable).  Differentiable once in q, k and v; two backward
    passes give the same bits.
    Tokens of a sequence from `max_seqlen` on are left out, with zeros for results and gradients; `check_attention` reports it."""
    q_strides = _rows("q", q)
    k_strides = _rows("k", k, like=q)
    v_strides = _rows("v", v, heads=k.shape[1], like=q)
    a = _problem(q, q_strides, k.shape[1], cu_seqlens, _host_int("max_seqlen", max_seqlen), _host_int("block", block),
                 _host_int("query_block", query_block, 1), causal)
    a.scale = _scale(scale, a.dim)
    _set_keys(a, k, k_strides, v, v_strides)
    _set_lists(a, lists, q.device)
    _on_gpu(q)
    return _BlockSparseAttention.apply(q, k, v, lists, cu_seqlens, a, return_lse)


def _report(status: torch.Tensor, name: str) -> None:
    """Raises what the kernels of any stream left in a status word, and clears it."""
    torch.cuda.synchronize(status.device)
    st = int(status.item())
    if st:
        status.zero_()
        torch.cuda.synchronize(status.device)    # no later call's report is cleared with this one's
        raise SpammError(st, name)


class _NoGradient(torch.autograd.Function):
    """A result without a gradient of its own, of tensors that want one: a backward pass through it raises."""

    @staticmethod
    def forward(ctx, x, source, name):
        ctx.name = name
        return x.view_as(x)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.name} has no gradient (block_sparse_attention has); run it under torch.no_grad() or on "
                           "detached tensors")


class PagedCache:
    """Keys and values of many sequences in pages of `page_size` tokens, with the sum of the keys of every page.

    k, v: [n_pages, kv_heads, page_size, head_dim]; key_sums: float [n_pages, kv_heads, head_dim] (zeros when not given: pages
    that hold keys already need theirs for `select`).  The caller hands out
    the pages: the page of tokens b * page_size .. of sequence s is page_table[s, b] (int32 [batch, width]), and
    lengths[s] (int32) tokens are held, counting the new ones of the call: the same two tensors serve `append`, `select`
    and `attend` of one step.

    What the tables say is checked on the GPU: a page outside the cache is read as masked and never written, tokens beyond
    the table's width, more new tokens than `max_new` or than the length holds are left out; `check()` reports any of these
    since the last report.  No two sequences may append to the same page in one call; reading a
    shared page is fine.

    The cache serves and does not train: a backward pass through a result of `append` or `attend`, when q or what was appended
    required gradients, raises RuntimeError."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, key_sums: Optional[torch.Tensor] = None):
        for name, x in (("k", k), ("v", v)):
            if not isinstance(x, torch.Tensor) or x.dim() != 4 or x.dtype not in _DTYPES or not x.is_contiguous():
                raise ValueError(f"{name} must be a contiguous bfloat16 or float16 tensor [n_pages, kv_heads, page_size, head_dim]")
        if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("k and v must match in shape, dtype and device")
        if k.shape[0] < 1 or k.shape[1] < 1 or k.shape[2] not in _BLOCKS or k.shape[3] not in (64, 128):
            raise ValueError(f"page size must be one of {_BLOCKS}, head_dim 64 or 128, got {tuple(k.shape)}")
        sums = (k.shape[0], k.shape[1], k.shape[3])
        if key_sums is not None and (key_sums.dtype != torch.float32 or tuple(key_sums.shape) != sums
                                     or key_sums.device != k.device or not key_sums.is_contiguous()):
            raise ValueError(f"key_sums must be a contiguous float32 tensor {sums} beside k")
        _on_gpu(k)
        self.k, self.v = k, v
        self.key_sums = torch.zeros(sums, dtype=torch.float32, device=k.device) if key_sums is None else key_sums
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._wanted_gradients = False           # some appended key or value did

    @classmethod
    def empty(cls, n_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, dtype=torch.bfloat16,
              device="cuda") -> "PagedCache":
        shape = (n_pages, kv_heads, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    def _without_gradient(self, x: torch.Tensor, q: torch.Tensor, name: str) -> torch.Tensor:
        if not torch.is_grad_enabled() or not (q.requires_grad or self._wanted_gradients):
            return x
        return _NoGradient.apply(x, q if q.requires_grad else torch.empty(0, requires_grad=True), "PagedCache." + name)

    def check(self) -> None:
        """Waits for the GPU (for the work of all streams) and raises SpammError when a call met a page, a length or a number
        of new tokens out of range since the last report."""
        _report(self.status, "PagedCache")

    def _problem(self, q, q_strides, cu_seqlens, max_new, page_table, lengths, query_block) -> SpammAttn:
        n_pages, kv_heads, page_size, dim = self.k.shape
        device = self.k.device
        if q.dtype != self.k.dtype or q.shape[2] != dim or q.device != device:
            raise ValueError("tokens must match the cache in dtype, head_dim and device")
        a = _problem(q, q_strides, kv_heads, cu_seqlens, _host_int("max_new", max_new), page_size,
                     _host_int("query_block", query_block, 1), True)
        batch = a.batch
        _ints("lengths", lengths, (batch,), device)
        if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2 or page_table.dtype != torch.int32 \
                or page_table.shape[0] != batch or page_table.device != device:
            raise ValueError("page_table must be an int32 tensor [batch, pages of the longest sequence] beside the tokens")
        width, (row, column) = page_table.shape[1], page_table.stride()
        if width > 1 and column != 1:
            raise ValueError("page_table: the last dimension must be contiguous")
        if batch > 1 and width and row < width:
            raise ValueError("page_table: rows must not overlap")
        a.n_pages = n_pages
        a.table_width = width
        a.table_stride = max(row, width) if batch > 1 else width
        a.d_table = page_table.data_ptr()
        a.d_lengths = lengths.data_ptr()
        a.d_status = self.status.data_ptr()
        return a

    def append(self, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, max_new: int, page_table: torch.Tensor,
               lengths: torch.Tensor, inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
               q: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Writes the new tokens' keys and values to their pages: token i of n new ones of sequence s to position
        lengths[s] - n + i.  With `inv_freq` (float32 [n], n a multiple of 8, 2 n <= head_dim) keys are rotated by
        position * inv_freq on the way, pairs (j, j + n) of each head or, `interleaved`, (2j, 2j + 1); `q` is rotated
        likewise and returned as a new tensor.  The key sums of the touched pages are taken anew from all keys that they
        hold, so that tokens may be appended again after `lengths` went back."""
        kv_heads = self.k.shape[1]
        k_strides = _rows("k", k, heads=kv_heads)
        v_strides = _rows("v", v, heads=kv_heads, like=k)
        q_strides = _rows("q", q, like=k) if q is not None else k_strides
        if inv_freq is not None:
            if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 \
                    or not inv_freq.is_contiguous() or inv_freq.device != k.device:
                raise ValueError("inv_freq must be a contiguous float32 tensor beside the tokens")
            if inv_freq.shape[0] % 8 or 2 * inv_freq.shape[0] > k.shape[2] or not inv_freq.shape[0]:
                raise ValueError(f"inv_freq must have a multiple of 8 values, at most head_dim / 2, got {inv_freq.shape[0]}")
        a = self._problem(k if q is None else q, q_strides, cu_seqlens, max_new, page_table, lengths, 1)
        _set_keys(a, k, k_strides, v, v_strides)
        if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
            self._wanted_gradients = True
        lib = _lib.load()
        with _device(k.device):
            out = None
            if q is not None:
                out = _like(q)
                _set_out(a, out)
                if not a.batch or not a.max_q:
                    out.zero_()
            check(lib.spamm_attn_append_dev(C.byref(a), self.k.data_ptr(), self.v.data_ptr(), self.key_sums.data_ptr(),
                                            inv_freq.data_ptr() if inv_freq is not None else None,
                                            inv_freq.shape[0] if inv_freq is not None else 0, int(bool(interleaved)),
                                            _stream(k.device)), "spamm_attn_append_dev")
        return self._without_gradient(out, q, "append") if q is not None else None

    def select(self, q: torch.Tensor, cu_seqlens: torch.Tensor, max_new: int, page_table: torch.Tensor, lengths: torch.Tensor,
               n_select: int, query_block: int = 1, n_first: int = 1, n_local: int = 1) -> torch.Tensor:
        """`select_blocks` for the newest tokens over the cached pages, by the cache's key sums."""
        a = self._problem(q, _rows("q", q), cu_seqlens, max_new, page_table, lengths, query_block)
        a.d_k = self.k.data_ptr()
        return _select(a, q, self.key_sums, _host_int("n_select", n_select, 1), _host_int("n_first", n_first),
                       _host_int("n_local", n_local))

    def attend(self, q: torch.Tensor, cu_seqlens: torch.Tensor, max_new: int, page_table: torch.Tensor, lengths: torch.Tensor,
               lists: Optional[torch.Tensor] = None, query_block: int = 1, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """Attention of the newest tokens (one of each sequence or a whole chunk) over the cached keys up to their own,
        of all pages or, with `lists` (as `select` gives them, for the same `query_block`), of the listed ones.  With
        `out` the result goes there, and its rows that belong to no sequence are left as they are; else they are zero.
        (As torch's own functions with an `out` it is refused where gradients are recorded for q or for `out`.)"""
        a = self._problem(q, _rows("q", q), cu_seqlens, max_new, page_table, lengths, query_block)
        if out is not None and torch.is_grad_enabled() and isinstance(out, torch.Tensor) and (q.requires_grad or out.requires_grad):
            raise ValueError("out: not where gradients are recorded (q or out requires them); call under torch.no_grad()")
        a.scale = _scale(scale, a.dim)
        a.d_k, a.d_v = self.k.data_ptr(), self.v.data_ptr()
        device = q.device
        if lists is not None:
            _set_lists(a, lists, device)
        with _device(device):
            if out is None:
                out = _like(q)
                if not a.batch or not a.max_q:
                    out.zero_()
                _set_out(a, out)
            else:
                a.o_token, a.o_head = _rows("out", out, heads=a.heads, like=q)
                if any(n > 1 and st == 0 for n, st in zip(out.shape, out.stride())):
                    raise ValueError("out: rows must not overlap")
                a.d_o = out.data_ptr()
                a.zero_tail = 0
            lse = None
            if return_lse:
                lse = torch.full((a.tokens, a.heads), float("-inf"), dtype=torch.float32, device=device)
                a.d_lse = lse.data_ptr()
            _forward(a, device)
        if a.zero_tail:
            out = self._without_gradient(out, q, "attend")
        if return_lse:
            lse = self._without_gradient(lse, q, "attend")
        return (out, lse) if return_lse else out
