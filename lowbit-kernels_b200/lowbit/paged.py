"""A paged KV cache and the two operators a chunk of new tokens runs against it: `norm_rope_append` (per-head norms of
q and k, rotary rotation, append to the cache in one pass) and `attention` (the new tokens of several sequences over
their cached contexts; one new token per sequence is a decode step). For drafted tokens that form trees: `plan` (page tables,
slots, positions and tree masks from lengths on the GPU), `tree_attention`, `verify` (which drafts are accepted) and `compact`
(their K and V rows move together). `PagedDecoder` runs them together with the 8-bit products of ops.linear_w8 and
ops.linear_f8. No counterpart in the reference, which feeds transformers' own cache (bench/e2e.py:84-147).

Every call launches on the current torch stream of the tensors' device and never synchronizes. Serving operators: their
outputs carry no autograd graph, whatever their inputs require. There is no fallback: without the library or a CUDA device
the first call raises.
"""
import collections
import ctypes
import math

import torch

from . import ops
from .decode import context_limit
from ._lib import DTYPE_IDS, PagedCacheStruct, _Device


class PagedCache:
    """K and V of one layer: [num_pages, nkv, page_size, hd] each, fp16 or bf16. Token j of a sequence lies in row
    j % page_size of page table[j // page_size]; the slot of a token is page * page_size + row. page_size is a multiple
    of 16; hd a multiple of 16 up to 256 (64 or 128 for `attention`). Which pages belong to whom is the caller's to
    keep; contents start undefined."""

    def __init__(self, num_pages, page_size, nkv, hd, dtype=torch.float16, device="cuda"):
        shape = (num_pages, nkv, page_size, hd)
        self._bind(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))

    @classmethod
    def from_tensors(cls, k, v):
        """Over existing tensors, without a copy; pages may be any multiple of 8 elements apart (k and v as halves of
        one [num_pages, 2, nkv, page_size, hd] tensor, say), each page's block contiguous."""
        self = cls.__new__(cls)
        self._bind(k, v)
        return self

    def _bind(self, k, v):
        if not (k.is_cuda and v.is_cuda and k.device == v.device):
            raise RuntimeError("the cache must be on one GPU")
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in (torch.float16, torch.bfloat16):
            raise RuntimeError("k and v must be float16 or bfloat16 [num_pages, nkv, page_size, hd] tensors of one shape")
        pages, nkv, page_size, hd = k.shape
        if page_size % 16 or not 16 <= page_size <= 65536:
            raise ValueError(f"page_size={page_size}: a multiple of 16 up to 65536")
        if hd % 16 or not 16 <= hd <= 256:
            raise ValueError(f"hd={hd}: head dims are multiples of 16 up to 256")
        if not k.numel():
            raise ValueError("the cache has no pages or no heads")
        for t in (k, v):
            if not t[0].is_contiguous() or (pages > 1 and (t.stride(0) % 8 or t.stride(0) < t[0].numel())):
                raise RuntimeError("each page's block must be contiguous, pages a multiple of 8 elements apart")
            if t.data_ptr() % 16:
                raise RuntimeError("the cache must be 16-byte aligned")
        block = k[0].numel()
        self._k, self._v, self._device = k, v, k.get_device()
        self.nkv, self.hd, self.page_size, self.num_pages, self.dtype = nkv, hd, page_size, pages, k.dtype
        self._struct = PagedCacheStruct(k.data_ptr(), v.data_ptr(), k.stride(0) if pages > 1 else block,
                                        v.stride(0) if pages > 1 else block, pages, DTYPE_IDS[k.dtype], nkv, hd, page_size)
        self._ptr = ctypes.addressof(self._struct)
        self._place = self._ptr, self._device

    @property
    def k(self):
        return self._k

    @property
    def v(self):
        return self._v


def _on(cache, name, t, dtype, *shape):
    """Raise unless t is a contiguous tensor of that type and shape (None: any) on the cache's GPU."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() == cache._device):
        raise RuntimeError(f"{name} must be on the cache's GPU, {cache.k.device}")
    if t.dtype != dtype or t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        raise RuntimeError(f"{name} must be a {dtype} {list(shape)} tensor, got {t.dtype} {list(t.shape)}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    return t.data_ptr()


def norm_rope_append(qkv, cache, positions, slots, nh, inv_freq, q_norm=None, k_norm=None, eps=1e-6, out=None):
    """One pass over the fused projection's rows qkv [T, (nh + 2 nkv) hd] of T new tokens (rows a multiple of 8 elements
    apart): q and k heads times rsqrt(mean(x^2) + eps) times q_norm / k_norm ([hd], both or neither), their first
    2 * len(inv_freq) dimensions rotated (rotate-half) by positions[t] * inv_freq (int64 [T], fp32), then k and v stored
    at the cache's slots (int64 [T]; negative: not stored; past the cache: not stored, and the device status becomes 3, as in
    `attention`). Returns q [T, nh, hd] (`out`, when given). All in fp32 with
    one rounding."""
    tc = ops._tc if ops._tc is not None else ops._torchcall()
    if tc:
        q = tc.norm_rope_append(qkv, cache._ptr, cache._device, positions, slots, nh, inv_freq, q_norm, k_norm, eps, out)
        if q is not None:
            return q
    if not (isinstance(qkv, torch.Tensor) and qkv.is_cuda and qkv.get_device() == cache._device):
        raise RuntimeError(f"qkv must be on the cache's GPU, {cache.k.device}")
    width = (nh + 2 * cache.nkv) * cache.hd
    if nh < 1 or qkv.dtype != cache.dtype or qkv.dim() != 2 or qkv.shape[1] != width:
        raise RuntimeError(f"qkv must be a {cache.dtype} [T, {width}] tensor, got {qkv.dtype} {list(qkv.shape)}")
    if qkv.stride(1) != 1 or (qkv.shape[0] > 1 and (qkv.stride(0) % 8 or qkv.stride(0) < width)) or qkv.data_ptr() % 16:
        raise RuntimeError("qkv rows must be contiguous, 16-byte aligned and a multiple of 8 elements apart")
    t = qkv.shape[0]
    pos, slot = _on(cache, "positions", positions, torch.int64, t), _on(cache, "slots", slots, torch.int64, t)
    freq = _on(cache, "inv_freq", inv_freq, torch.float32, None)
    rot = 2 * inv_freq.numel()
    if rot % 16 or rot > cache.hd:
        raise RuntimeError(f"inv_freq holds half of the rotated dimensions, a multiple of 8 up to hd / 2 = {cache.hd // 2}")
    if (q_norm is None) != (k_norm is None):
        raise RuntimeError("q_norm and k_norm go together")
    qn = None if q_norm is None else _on(cache, "q_norm", q_norm, cache.dtype, cache.hd)
    kn = None if k_norm is None else _on(cache, "k_norm", k_norm, cache.dtype, cache.hd)
    if out is None:
        out = torch.empty(t, nh, cache.hd, dtype=cache.dtype, device=qkv.device)
    _on(cache, "out", out, cache.dtype, t, nh, cache.hd)
    if t == 0:
        return out
    e = ops.ext()
    with _Device(qkv.device):
        rc = e.lib.lb_paged_norm_rope_append(qkv.data_ptr(), qkv.stride(0) if t > 1 else width, t, nh, qn, kn, eps,
                                             freq if rot else None, rot, pos, slot, cache._ptr, out.data_ptr(),
                                             torch.cuda.current_stream().cuda_stream)
    if rc:
        e._raise(rc)
    return out


def attention(q, cache, page_table, seq_lens, cu_new, max_new=None, max_len=None, scale=None, out=None):
    """Attention of new tokens over the paged cache that already holds them. q [T, nh, hd] (heads and tokens a multiple
    of 8 elements apart); sequence s has the tokens cu_new[s] .. cu_new[s + 1] - 1 (int32 [S + 1], from 0) and, them
    included, seq_lens[s] tokens (int32 [S]) in the pages page_table[s] (int32 [S, W]); its new token i of n sees keys
    0 .. seq_lens[s] - n + i, none giving zeros. Query heads share key heads in groups of nh / nkv. Returns [T, nh, hd].

    max_new and max_len bound the new tokens and the context of any sequence (host integers; by default T and
    W * page_size). They choose the kernel and how contexts are split, so a decode step passes max_new=1; a bound below
    the truth is an error that leaves outputs undefined. A page-table entry outside the cache counts as a page of zeros and
    sets the library's device status to 3 (`ops.ext().lib.lb_device_error()`, which synchronizes; no call reads it by
    itself). scale defaults to 1 / sqrt(hd). Cache rows past a context may hold anything; inside one, a V row with an
    infinity or NaN can make earlier new tokens of the call NaN too, as 0 times it does. Tokens past cu_new[S] (a padded
    batch's) belong to no sequence: their outputs are left unwritten."""
    tc = ops._tc if ops._tc is not None else ops._torchcall()
    if tc:
        y = tc.paged_attention(q, cache._ptr, cache._device, page_table, seq_lens, cu_new, max_new, max_len, scale, out)
        if y is not None:
            return y
    return _attend(q, cache, page_table, seq_lens, cu_new, None, max_new, max_len, scale, out)


def tree_attention(q, cache, page_table, seq_lens, cu_new, mask, max_new=None, max_len=None, scale=None, out=None):
    """`attention` for drafted tokens that form trees. mask int32 [T, words]: bit j % 32 of word j / 32 of a token's row says
    whether it sees its sequence's new token j (`plan` makes it from the tokens' parents; any pattern will do, a row of zeros
    too). Every new token sees the whole cached context, the keys before the sequence's new ones, which lie in the cache in the
    order of the call; new tokens past 32 * words are seen by none. A V row with an infinity or NaN can make any new token of the same
    call NaN, whether it sees that row or not. The rest is as in `attention`."""
    tc = ops._tc if ops._tc is not None else ops._torchcall()
    if tc:
        y = tc.paged_tree_attention(q, cache._ptr, cache._device, page_table, seq_lens, cu_new, mask, max_new, max_len, scale, out)
        if y is not None:
            return y
    if mask is None:
        raise RuntimeError("mask must be an int32 [T, words] tensor on the cache's GPU")
    return _attend(q, cache, page_table, seq_lens, cu_new, mask, max_new, max_len, scale, out)


def _attend(q, cache, page_table, seq_lens, cu_new, mask, max_new, max_len, scale, out):
    """The checked path of both attentions; mask: a tree's, or None."""
    if not (isinstance(q, torch.Tensor) and q.is_cuda and q.get_device() == cache._device):
        raise RuntimeError(f"q must be on the cache's GPU, {cache.k.device}")
    if q.dtype != cache.dtype or q.dim() != 3 or q.shape[2] != cache.hd:
        raise RuntimeError(f"q must be a {cache.dtype} [T, nh, {cache.hd}] tensor, got {q.dtype} {list(q.shape)}")
    t, nh, hd = q.shape
    if cache.hd not in (64, 128):
        raise RuntimeError(f"hd={hd}: the attention takes head dims 64 and 128")
    if nh == 0 or nh % cache.nkv:
        raise RuntimeError(f"nh={nh} must be a multiple of nkv={cache.nkv}")
    t_stride, h_stride = q.stride(0) if t > 1 else 0, q.stride(1) if nh > 1 else 0
    if q.stride(2) != 1 or t_stride % 8 or h_stride % 8 or q.data_ptr() % 16:
        raise RuntimeError("q's heads must be contiguous, 16-byte aligned, heads and tokens a multiple of 8 elements apart")
    if not (isinstance(page_table, torch.Tensor) and page_table.is_cuda and page_table.get_device() == cache._device
            and page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.shape[1] > 0
            and page_table.stride(1) == 1):
        raise RuntimeError("page_table must be an int32 [S, W] tensor on the cache's GPU, its rows contiguous")
    s, width = page_table.shape
    lens, cu = _on(cache, "seq_lens", seq_lens, torch.int32, s), _on(cache, "cu_new", cu_new, torch.int32, s + 1)
    if out is None:
        out = torch.empty(t, nh, hd, dtype=q.dtype, device=q.device)
    _on(cache, "out", out, cache.dtype, t, nh, hd)
    if mask is not None:
        bits = _on(cache, "mask", mask, torch.int32, t, None)
        if mask.shape[1] < 1:
            raise RuntimeError("mask must have a word a row at least")
    max_new = t if max_new is None else int(max_new)
    max_len = width * cache.page_size if max_len is None else int(max_len)
    if t == 0 or s == 0:
        return out
    e = ops.ext()
    with _Device(q.device):
        space = e.lib.lb_paged_attention_workspace if mask is None else e.lib.lb_paged_tree_attention_workspace
        need = space(t, nh, cache._ptr, width, s, max_new, max_len)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        head = (q.data_ptr(), t_stride, h_stride, t, nh, cache._ptr, page_table.data_ptr(),
                page_table.stride(0) if s > 1 else width, width, lens, cu, s)
        tail = (max_new, max_len, 1 / math.sqrt(hd) if scale is None else scale, out.data_ptr(), nh * hd,
                ws.data_ptr() if need else None, need, torch.cuda.current_stream().cuda_stream)
        if mask is None:
            rc = e.lib.lb_paged_attention(*head, *tail)
        else:
            rc = e.lib.lb_paged_tree_attention(*head, bits, mask.shape[1], *tail)
    if rc:
        e._raise(rc)
    return out


Plan = collections.namedtuple("Plan", "cu_new seq_lens positions slots held free_count mask")
Plan.__doc__ = """What `plan` gives: cu_new int32 [S + 1], seq_lens int32 [S] (the tokens with the new ones; 0: refused), positions and
slots int64 [tokens], held int32 [S] and free_count int32 [1] (None without pages to give out), mask int32 [tokens, words] (None
without parents)."""
Verified = collections.namedtuple("Verified", "accepted path next targets")
Verified.__doc__ = """What `verify` gives: accepted int32 [S], path int32 [S, max_path], next int64 [S], targets int64 [T]."""


def _vector(name, t, dtype, device, *shape):
    """Raise unless t is a contiguous tensor of that type and shape (None: any) on that GPU; its address."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.device == device):
        raise RuntimeError(f"{name} must be on {device}")
    if t.dtype != dtype or t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        raise RuntimeError(f"{name} must be a {dtype} {list(shape)} tensor, got {t.dtype} {list(t.shape)}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    return t.data_ptr()


def _page_table(t):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.int32 and t.dim() == 2 and t.shape[0] > 0
            and t.shape[1] > 0 and t.stride(1) == 1):
        raise RuntimeError("page_table must be an int32 [S, W] tensor on the GPU, its rows contiguous")
    s, width = t.shape
    if s > 1 and t.stride(0) < width:
        raise RuntimeError("page_table's rows overlap")
    return s, width, t.stride(0) if s > 1 else width


def plan(page_table, seq_lens, new_lens, page_size, tokens, held=None, free_pages=None, free_count=None, parents=None,
         max_new=None, out=None):
    """What a call on new tokens needs, built on the GPU: sequence s has seq_lens[s] tokens in the cache and gets new_lens[s]
    more (int32 [S] each, S up to 8192). Returns a `Plan` whose rows are the sequences' new tokens one after another, `tokens`
    of them (a host integer, at least their sum); rows past the last sequence get position 0 and slot -1, so that
    `norm_rope_append` stores nothing for them and `attention` leaves them out.

    held int32 [S], free_pages int32 [P] and free_count int32 [1], all or none, let it give out pages: row s of page_table int32
    [S, W] holds held[s] pages, and what the new tokens need beyond them is taken from the first free_count[0] entries of free_pages,
    the last first, by the sequences in their order, and written into page_table behind them; the plan's held and free_count say
    what there is then. Without them page_table is complete as it is. A sequence is refused where `tokens`, W or the free pages do not suffice
    (from the first that lacks pages on, all that need some), or where it is a tree of more tokens than its mask has bits: its seq_lens is
    0, so that attention gives it zeros (its rows past the attention's max_new are left unwritten), its slots are -1, and it takes no pages.

    parents int32 [tokens]: the new tokens of a sequence form a tree, parents[t] being the place among them of the token's
    parent, an earlier one; anything else makes it a root. Positions are then seq_lens + depth, and the plan's mask is what
    `tree_attention` takes, its rows ceil(max_new / 32) words (max_new bounds the new tokens of any sequence, 1024 at most; by default
    tokens). A tree is refused by the mask's bits: one of more than max_new tokens that they hold is served, and then `tree_attention` and
    `verify`, for which max_new has to be the truth, need 32 * mask.shape[1]. Where lengths may pass the bound all three take a multiple of 32.

    out: a Plan whose tensors receive the result (fixed addresses for a captured step); its held, free_count and seq_lens may be the
    ones passed in, nothing else of it may lie over an input. Without it the tensors of a result may share one allocation: one that is
    kept or saved keeps all of it, its clone() does not."""
    tc = ops._tc if ops._tc is not None else ops._torchcall()
    if tc and out is None:
        got = tc.plan(page_table, seq_lens, new_lens, page_size, tokens, held, free_pages, free_count, parents, max_new)
        if got is not None:
            return Plan._make(got)
    s, width, stride = _page_table(page_table)
    dev = page_table.device
    lens, new = _vector("seq_lens", seq_lens, torch.int32, dev, s), _vector("new_lens", new_lens, torch.int32, dev, s)
    paging = held is not None
    if paging != (free_pages is not None) or paging != (free_count is not None):
        raise RuntimeError("held, free_pages and free_count go together")
    tokens = int(tokens)
    words = 0
    if parents is not None:
        max_new = tokens if max_new is None else int(max_new)
        words = -(-max(1, max_new) // 32)
        if words > 32:
            raise ValueError(f"max_new={max_new}: trees hold up to 1024 tokens")
    if out is None:
        def make(dtype, *shape):
            return torch.empty(shape, dtype=dtype, device=dev)
        out = Plan(make(torch.int32, s + 1), make(torch.int32, s), make(torch.int64, tokens), make(torch.int64, tokens),
                   make(torch.int32, s) if paging else None, make(torch.int32, 1) if paging else None,
                   make(torch.int32, tokens, words) if words else None)
    cu, after = _vector("out.cu_new", out.cu_new, torch.int32, dev, s + 1), _vector("out.seq_lens", out.seq_lens, torch.int32, dev, s)
    pos, slots = (_vector(f"out.{n}", t, torch.int64, dev, tokens) for n, t in (("positions", out.positions), ("slots", out.slots)))
    pages = [None, None, 0, None, None, None]
    if paging:
        pages = [_vector("held", held, torch.int32, dev, s), _vector("free_pages", free_pages, torch.int32, dev, None), free_pages.numel(),
                 _vector("free_count", free_count, torch.int32, dev, 1), _vector("out.held", out.held, torch.int32, dev, s),
                 _vector("out.free_count", out.free_count, torch.int32, dev, 1)]
    tree = bits = None
    if words:
        tree = _vector("parents", parents, torch.int32, dev, tokens)
        bits = _vector("out.mask", out.mask, torch.int32, dev, tokens, words)
        if not tokens:   # (an empty tensor has no address)
            tree = bits = None
    e = ops.ext()
    with _Device(dev):
        rc = e.lib.lb_paged_plan(lens, new, s, page_table.data_ptr(), stride, width, int(page_size), tokens, pages[0], pages[1] or (lens if paging else None),
                                 pages[2], pages[3], tree, words if tree else 0, cu, after, pages[4], pages[5], pos, slots, bits,
                                 torch.cuda.current_stream().cuda_stream)
    if rc:
        e._raise(rc)
    return out


def verify(logits, tokens, parents, cu_new, max_new=None, max_path=None, seq_lens=None):
    """Greedy acceptance of drafted trees. logits [T, vocab] (fp16, bf16 or fp32, rows any stride apart) follow the new tokens
    `tokens` int64 [T] of the sequences cu_new int32 [S + 1], whose parents int32 [T] are as in `plan`. Returns a `Verified`: targets,
    the index of each row's first largest value (a NaN counts as larger than all); and for each sequence the path that starts at its first new token, the
    last certain one, and goes on to the first later token that is a child of the one at hand and equals its target: how many tokens it has
    (accepted), their places among the new ones (path, -1 behind them) and the target after the last (next). A sequence
    without new tokens gets 0 and -1. max_new bounds the new tokens of any sequence (1024 at most; by default T;
    those past it are left out, their targets unwritten), max_path the path (by default max_new). Rows past cu_new[S] are not looked at, their targets left unwritten.

    A sequence that `plan` refused may have rows, and the logits after them come from tokens that saw nothing. With the plan's seq_lens
    (int32 [S]) it gets 0 and -1 too; without them its path and next mean nothing, and the caller looks at the plan's seq_lens before
    using them. The four tensors, and the call's scratch memory, may share one allocation."""
    tc = ops._tc if ops._tc is not None else ops._torchcall()
    if tc:
        got = tc.verify(logits, tokens, parents, cu_new, max_new, max_path, seq_lens)
        if got is not None:
            return Verified._make(got)
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dim() == 2 and logits.dtype in DTYPE_IDS):
        raise RuntimeError("logits must be a float16, bfloat16 or float32 [T, vocab] tensor on the GPU")
    t, vocab = logits.shape
    if not vocab:
        raise RuntimeError("the vocabulary is empty")
    if logits.stride(1) != 1 and vocab > 1 or t > 1 and logits.stride(0) < vocab:
        logits = logits.contiguous()
    dev = logits.device
    drafted, tree = _vector("tokens", tokens, torch.int64, dev, t), _vector("parents", parents, torch.int32, dev, t)
    cu = _vector("cu_new", cu_new, torch.int32, dev, None)
    s = cu_new.numel() - 1
    if s < 1:
        raise RuntimeError("cu_new must hold a sequence at least")
    lens = None if seq_lens is None else _vector("seq_lens", seq_lens, torch.int32, dev, s)
    max_new = t if max_new is None else int(max_new)
    max_path = max_new if max_path is None else int(max_path)
    if t and not 1 <= max_new <= 1024:
        raise ValueError(f"max_new={max_new}: trees hold 1 to 1024 tokens")
    if t and not 1 <= max_path <= 1024:
        raise ValueError(f"max_path={max_path}: 1 to 1024")
    if t == 0:
        return Verified(torch.zeros(s, dtype=torch.int32, device=dev), torch.full((s, max(1, max_path)), -1, dtype=torch.int32, device=dev),
                        torch.full((s,), -1, dtype=torch.int64, device=dev), torch.empty(0, dtype=torch.int64, device=dev))
    got = Verified(torch.empty(s, dtype=torch.int32, device=dev), torch.empty(s, max_path, dtype=torch.int32, device=dev),
                   torch.empty(s, dtype=torch.int64, device=dev), torch.empty(t, dtype=torch.int64, device=dev))
    e = ops.ext()
    with _Device(dev):
        need = e.lib.lb_draft_verify_workspace(t, vocab)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        rc = e.lib.lb_draft_verify_planned(logits.data_ptr(), DTYPE_IDS[logits.dtype], logits.stride(0) if t > 1 else vocab, t, vocab, drafted,
                                           tree, cu, lens, s, max_new, max_path, got.accepted.data_ptr(), got.path.data_ptr(), got.next.data_ptr(),
                                           got.targets.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    if rc:
        e._raise(rc)
    return got


def compact(caches, page_table, seq_lens, cu_new, path, accepted, out=None):
    """Moves the accepted tokens' K and V rows to where a sequence without the other drafts has them, in all of `caches` (a list
    of up to 128 PagedCache of one layout, a layer each, none twice): with n new tokens of sequence s and seq_lens[s] tokens, them
    included, row seq_lens[s] - n + path[s, d] goes to seq_lens[s] - n + d for d < accepted[s] (path int32 [S, D] and accepted
    int32 [S] as `verify` gives them: a path rises). Returns seq_lens[s] - n + accepted[s], int32 [S] (`out`, when given: over
    none of the inputs). For a sequence that `plan` refused (its seq_lens is 0, whether it has rows or not), and for an empty one,
    this is 0, or what `out` held, and nothing moves: with the lengths before the plan as `out` a refused sequence keeps its
    context. A path's entry outside the new tokens, below its own place, or on a page outside the cache is left out, and the
    device status becomes 3, as in `attention`; whether it rises is not looked at, an entry that does not is moved as it stands."""
    tc = ops._tc if ops._tc is not None else ops._torchcall()
    if tc:
        got = tc.compact(caches, PagedCache, page_table, seq_lens, cu_new, path, accepted, out)
        if got is not None:
            return got
    caches = list(caches)
    if not caches or not all(isinstance(c, PagedCache) for c in caches):
        raise RuntimeError("caches must be a list of PagedCache")
    cache = caches[0]
    if any(c._device != cache._device for c in caches):
        raise RuntimeError("the caches must be on one GPU")
    s, width, stride = _page_table(page_table)
    if page_table.get_device() != cache._device:
        raise RuntimeError(f"page_table must be on the cache's GPU, {cache.k.device}")
    lens, cu = _on(cache, "seq_lens", seq_lens, torch.int32, s), _on(cache, "cu_new", cu_new, torch.int32, s + 1)
    at, count = _on(cache, "path", path, torch.int32, s, None), _on(cache, "accepted", accepted, torch.int32, s)
    keep = out is not None
    if not keep:
        out = torch.empty(s, dtype=torch.int32, device=page_table.device)
    dst = _on(cache, "out", out, torch.int32, s)
    e = ops.ext()
    with _Device(page_table.device):
        rc = e.lib.lb_paged_compact((ctypes.c_void_p * len(caches))(*[c._ptr for c in caches]), len(caches), page_table.data_ptr(), stride,
                                    width, lens, cu, at, count, s, path.shape[1], dst, keep, torch.cuda.current_stream().cuda_stream)
    if rc:
        e._raise(rc)
    return out


class PagedDecoder:
    """A Qwen2-architecture decoder whose calls take chunks of new tokens of any number of sequences -- a prompt in
    pieces, single tokens of a running batch, or both at once -- over paged caches. Takes the weights of a transformers
    model of that architecture (fp16 or bf16; per-head q_norm / k_norm modules are used where its attention has them)
    and keeps its projections in 8-bit integers (`weights="w8"`, ops.linear_w8), in 8-bit floating point with block scales
    (`weights="f8"`, ops.linear_f8) or, fp16 models only, in the INT4 format (`weights="w4"`, ops.linear). Per layer: RMSNorm, the fused q|k|v product, `norm_rope_append`, `attention`, the output
    product, RMSNorm, the fused gate|up product, SiLU * up, the down product. Models that scale their rotary angles, with an
    activation other than SiLU or with head dims other than 64 and 128 are refused (ValueError); one whose attention slides
    over a window, or whose angles are scaled only from some length on, takes contexts up to that length.

        dec = PagedDecoder(model, num_pages=512, page_size=64)
        a, b = dec.open(), dec.open()
        logits = dec.forward({a: prompt_a, b: prompt_b[:512]})      # [2, vocab]: after each chunk's last token
        logits = dec.forward({a: [next_a], b: prompt_b[512:]})
        more = dec.verify({a: ([next_a, x, y, z], [-1, 0, 0, 1])})   # drafts x and y after next_a, z after x
        dec.close(a)
    """

    def __init__(self, model, num_pages, page_size=64, weights="w8", group=128):
        if weights not in ("w8", "f8", "w4"):
            raise ValueError('weights is "w8", "f8" or "w4"')
        cfg, base = model.config, model.model
        self.limit = context_limit(cfg)
        self.embed = base.embed_tokens.weight.detach()
        self.device, self.dtype = self.embed.device, self.embed.dtype
        if weights == "w4" and self.dtype != torch.float16:
            raise ValueError("INT4 weights need a float16 model")
        self.nh, self.nkv = cfg.num_attention_heads, cfg.num_key_value_heads
        self.hd = getattr(cfg, "head_dim", None) or cfg.hidden_size // self.nh
        if self.hd not in (64, 128):
            raise ValueError(f"hd={self.hd}: the attention takes head dims 64 and 128")
        self.eps, self.page_size, self.vocab = float(cfg.rms_norm_eps), page_size, cfg.vocab_size
        theta = float(cfg.rope_parameters["rope_theta"])
        half = torch.arange(0, self.hd, 2, dtype=torch.float32)
        self.inv_freq = (1.0 / theta ** (half / self.hd)).to(self.device)
        if weights == "w8":
            self._make, self._linear = ops.W8Weight.from_float, ops.linear_w8
        elif weights == "f8":
            self._make, self._linear = ops.F8Weight.from_float, ops.linear_f8
        else:
            self._make = lambda w: ops.W4Weight.from_float(w, group, ("mma",))
            self._linear = ops.linear

        def vector(module):
            return None if module is None else module.weight.detach().to(self.dtype).contiguous()

        def fused(*linears):
            biases = [lin.bias for lin in linears]
            bias = None if biases[0] is None else torch.cat([b.detach() for b in biases]).to(self.dtype).contiguous()
            return self._make(torch.cat([lin.weight.detach() for lin in linears])), bias

        self.layers = []
        for layer in base.layers:
            a, m = layer.self_attn, layer.mlp
            self.layers.append({
                "qkv": fused(a.q_proj, a.k_proj, a.v_proj), "o": fused(a.o_proj), "gate_up": fused(m.gate_proj, m.up_proj),
                "down": fused(m.down_proj), "ln1": vector(layer.input_layernorm), "ln2": vector(layer.post_attention_layernorm),
                "q_norm": vector(getattr(a, "q_norm", None)), "k_norm": vector(getattr(a, "k_norm", None)),
                "cache": PagedCache(num_pages, page_size, self.nkv, self.hd, dtype=self.dtype, device=self.device)})
        self.norm, self.head = vector(base.norm), model.lm_head.weight.detach()
        self._free = list(range(num_pages - 1, -1, -1))
        self._seqs, self._next = {}, 0

    def open(self):
        """A new empty sequence's id."""
        sid, self._next = self._next, self._next + 1
        self._seqs[sid] = {"length": 0, "pages": []}
        return sid

    def close(self, sid):
        """Forget a sequence; its pages are free for others."""
        self._free += reversed(self._seqs.pop(sid)["pages"])

    def _rms(self, x, w):
        f = x.float()
        return w * (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + self.eps)).to(self.dtype)

    def _plan(self, chunks, reach=None):
        """The call's host arrays -- token ids, positions and slots, page table, lengths and first tokens -- and each
        sequence's pages after it. reach: how many tokens each sequence's context grows by, where its new ones do not follow one another
        (a tree's levels). Changes nothing: `_commit` does, once the call's work is launched."""
        page = self.page_size
        longest = max(self._seqs[s]["length"] + (len(new) if reach is None else reach[s]) for s, new in chunks.items())
        if self.limit is not None and longest > self.limit:
            raise ValueError(f"{longest} tokens: the model's sliding window or rotary scaling allows {self.limit} here")
        need = {s: -(-(self._seqs[s]["length"] + len(new)) // page) - len(self._seqs[s]["pages"]) for s, new in chunks.items()}
        if sum(need.values()) > len(self._free):
            raise RuntimeError(f"{sum(need.values())} pages are needed, {len(self._free)} are free")
        ids, pos, slots, lens, cu, pages, taken = [], [], [], [], [0], {}, 0
        for s, new in chunks.items():
            start = self._seqs[s]["length"]
            pages[s] = self._seqs[s]["pages"] + [self._free[-1 - taken - i] for i in range(need[s])]
            taken += need[s]
            for i, tok in enumerate(new, start):
                tok = int(tok)
                if not 0 <= tok < self.embed.shape[0]:   # (on the GPU the lookup's own check would end the context)
                    raise ValueError(f"token id {tok} of {self.embed.shape[0]}")
                ids.append(tok)
                pos.append(i)
                slots.append(pages[s][i // page] * page + i % page)
            lens.append(start + len(new))
            cu.append(len(ids))
        width = max(1, max(len(v) for v in pages.values()))
        table = [v + [0] * (width - len(v)) for v in pages.values()]
        return ids, pos, slots, table, lens, cu, pages

    def _commit(self, pages, lens):
        """The sequences hold those pages and that many tokens."""
        taken = sum(len(v) - len(self._seqs[s]["pages"]) for s, v in pages.items())
        del self._free[len(self._free) - taken:]
        for (s, v), n in zip(pages.items(), lens):
            self._seqs[s] = {"length": n, "pages": v}

    def _layers(self, x, pos, slots, attend):
        """The residual stream x [T, hidden] after all layers; attend(q, cache) is their attention."""
        for ly in self.layers:
            def product(h, name):
                w, bias = ly[name]
                return self._linear(h, w, bias=bias)
            qkv = product(self._rms(x, ly["ln1"]), "qkv")
            q = norm_rope_append(qkv, ly["cache"], pos, slots, self.nh, self.inv_freq, ly["q_norm"], ly["k_norm"], self.eps)
            x = x + product(attend(q, ly["cache"]).view(len(x), self.nh * self.hd), "o")
            gate, up = product(self._rms(x, ly["ln2"]), "gate_up").chunk(2, -1)
            x = x + product(torch.nn.functional.silu(gate) * up, "down")
        return x

    @torch.no_grad()
    def forward(self, chunks):
        """chunks: {sequence id: its new token ids, at least one}. Appends them and returns the logits [len(chunks),
        vocab] after each sequence's last new token, in the order of `chunks`. A call that raises (ValueError for
        a token id outside the embedding) leaves every sequence and the free pages as they were."""
        if not chunks or any(len(new) == 0 for new in chunks.values()):
            raise ValueError("every sequence of a call needs a new token")
        ids, pos, slots, table, lens, cu, pages = self._plan(chunks)
        dev = self.device
        ids, pos, slots = (torch.tensor(v, dtype=torch.int64, device=dev) for v in (ids, pos, slots))
        table, lens_d, cu_d = (torch.tensor(v, dtype=torch.int32, device=dev) for v in (table, lens, cu))
        max_new, max_len = max(len(new) for new in chunks.values()), max(lens)
        x = self._layers(self.embed[ids], pos, slots,
                         lambda q, cache: attention(q, cache, table, lens_d, cu_d, max_new=max_new, max_len=max_len))
        last = torch.tensor([c - 1 for c in cu[1:]], dtype=torch.int64, device=dev)
        logits = torch.nn.functional.linear(self._rms(x[last], self.norm), self.head)
        self._commit(pages, lens)
        return logits

    @torch.no_grad()
    def verify(self, trees):
        """trees: {sequence id: (tokens, parents)}. A sequence's first token is its last certain one, not fed yet (what `forward` or
        `verify` gave as the next), its parent -1; each further one is a draft that follows the token at its parent's place,
        an earlier one. All of them run through the model at once. Returns {sequence id: its new certain tokens}, one at least:
        the drafts on the path that the model's own choices (the first largest logit) take from the first token, then its choice after the
        last of them, which is the first token of the next call. The sequences keep the first token and the accepted drafts. A call
        that raises (ValueError for a token id outside the embedding or parents that are no tree) leaves every sequence and the
        free pages as they were."""
        if not trees:
            raise ValueError("no trees")
        levels = {}
        for s, (tokens, parents) in trees.items():
            if not 1 <= len(tokens) <= 1024 or len(parents) != len(tokens):
                raise ValueError("a tree has 1 to 1024 tokens, and a parent for each")
            if int(parents[0]) != -1 or any(not 0 <= int(p) < i for i, p in enumerate(parents[1:], 1)):
                raise ValueError("the first token's parent is -1, any other's an earlier token's place")
            depth = [1]
            for p in parents[1:]:
                depth.append(depth[int(p)] + 1)
            levels[s] = max(depth)   # what the longest path adds to the context; the branches beside it see none of each other
        ids, _, _, table, lens, cu, pages = self._plan({s: tokens for s, (tokens, _) in trees.items()}, levels)
        dev, new = self.device, [b - a for a, b in zip(cu, cu[1:])]
        drafted = torch.tensor(ids, dtype=torch.int64, device=dev)
        ints = (table, [n - k for n, k in zip(lens, new)], new, [int(p) for _, parents in trees.values() for p in parents])
        table_d, before, new_d, parents = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ints)
        max_new, max_len = max(new), max(lens)
        at = plan(table_d, before, new_d, self.page_size, len(ids), parents=parents, max_new=max_new)
        x = self._layers(self.embed[drafted], at.positions, at.slots,
                         lambda q, cache: tree_attention(q, cache, table_d, at.seq_lens, at.cu_new, at.mask, max_new=max_new, max_len=max_len))
        logits = torch.nn.functional.linear(self._rms(x, self.norm), self.head)
        got = verify(logits, drafted, parents, at.cu_new, max_new=max_new)
        caches = [ly["cache"] for ly in self.layers]
        for i in range(0, len(caches), 128):   # (as many as a call takes)
            compact(caches[i:i + 128], table_d, at.seq_lens, at.cu_new, got.path, got.accepted)
        accepted, path, following = got.accepted.tolist(), got.path.tolist(), got.next.tolist()
        kept = [n - k + a for n, k, a in zip(lens, new, accepted)]
        self._commit(pages, kept)
        more = {}
        for (s, (tokens, _)), a, way, nxt in zip(trees.items(), accepted, path, following):
            mine, need = self._seqs[s]["pages"], -(-self._seqs[s]["length"] // self.page_size)
            self._free += reversed(mine[need:])
            del mine[need:]
            more[s] = [int(tokens[i]) for i in way[1:a]] + [nxt]
        return more
