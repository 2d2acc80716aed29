"""A paged KV cache and the two operators a chunk of new tokens runs against it: `norm_rope_append` (per-head norms of
q and k, rotary rotation, append to the cache in one pass) and `attention` (the new tokens of several sequences over
their cached contexts; one new token per sequence is a decode step). `PagedDecoder` runs them together with the 8-bit
products of ops.linear_w8. No counterpart in the reference, which feeds transformers' own cache (bench/e2e.py:84-147).

Every call launches on the current torch stream of the tensors' device and never synchronizes. Serving operators: their
outputs carry no autograd graph, whatever their inputs require. There is no fallback: without the library or a CUDA device
the first call raises.
"""
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
    max_new = t if max_new is None else int(max_new)
    max_len = width * cache.page_size if max_len is None else int(max_len)
    if t == 0 or s == 0:
        return out
    e = ops.ext()
    with _Device(q.device):
        need = e.lib.lb_paged_attention_workspace(t, nh, cache._ptr, width, s, max_new, max_len)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        rc = e.lib.lb_paged_attention(q.data_ptr(), t_stride, h_stride, t, nh, cache._ptr, page_table.data_ptr(),
                                      page_table.stride(0) if s > 1 else width, width, lens, cu, s, max_new, max_len,
                                      1 / math.sqrt(hd) if scale is None else scale, out.data_ptr(), nh * hd,
                                      ws.data_ptr() if need else None, need,
                                      torch.cuda.current_stream().cuda_stream)
    if rc:
        e._raise(rc)
    return out


class PagedDecoder:
    """A Qwen2-architecture decoder whose calls take chunks of new tokens of any number of sequences -- a prompt in
    pieces, single tokens of a running batch, or both at once -- over paged caches. Takes the weights of a transformers
    model of that architecture (fp16 or bf16; per-head q_norm / k_norm modules are used where its attention has them)
    and keeps its projections in 8-bit integers (`weights="w8"`, ops.linear_w8) or, fp16 models only, in the INT4 format
    (`weights="w4"`, ops.linear). Per layer: RMSNorm, the fused q|k|v product, `norm_rope_append`, `attention`, the output
    product, RMSNorm, the fused gate|up product, SiLU * up, the down product. Models that scale their rotary angles, with an
    activation other than SiLU or with head dims other than 64 and 128 are refused (ValueError); one whose attention slides
    over a window, or whose angles are scaled only from some length on, takes contexts up to that length.

        dec = PagedDecoder(model, num_pages=512, page_size=64)
        a, b = dec.open(), dec.open()
        logits = dec.forward({a: prompt_a, b: prompt_b[:512]})      # [2, vocab]: after each chunk's last token
        logits = dec.forward({a: [next_a], b: prompt_b[512:]})
        dec.close(a)
    """

    def __init__(self, model, num_pages, page_size=64, weights="w8", group=128):
        if weights not in ("w8", "w4"):
            raise ValueError('weights is "w8" or "w4"')
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

    def _plan(self, chunks):
        """The call's host arrays -- token ids, positions and slots, page table, lengths and first tokens -- and each
        sequence's pages after it. Changes nothing: `_commit` does, once the call's work is launched."""
        page = self.page_size
        longest = max(self._seqs[s]["length"] + len(new) for s, new in chunks.items())
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

    @torch.no_grad()
    def forward(self, chunks):
        """chunks: {sequence id: its new token ids, at least one}. Appends them and returns the logits [len(chunks),
        vocab] after each sequence's last new token, in the order of `chunks`. A call that raises (ValueError for
        a token id outside the embedding) leaves every sequence and the free pages as they were."""
        if not chunks or any(len(new) == 0 for new in chunks.values()):
            raise ValueError("every sequence of a call needs a new token")
        ids, pos, slots, table, lens, cu, pages = self._plan(chunks)
        dev, t = self.device, len(ids)
        ids, pos, slots = (torch.tensor(v, dtype=torch.int64, device=dev) for v in (ids, pos, slots))
        table, lens_d, cu_d = (torch.tensor(v, dtype=torch.int32, device=dev) for v in (table, lens, cu))
        max_new, max_len = max(len(new) for new in chunks.values()), max(lens)
        x = self.embed[ids]
        for ly in self.layers:
            def product(h, name):
                w, bias = ly[name]
                return self._linear(h, w, bias=bias)
            qkv = product(self._rms(x, ly["ln1"]), "qkv")
            q = norm_rope_append(qkv, ly["cache"], pos, slots, self.nh, self.inv_freq, ly["q_norm"], ly["k_norm"], self.eps)
            a = attention(q, ly["cache"], table, lens_d, cu_d, max_new=max_new, max_len=max_len)
            x = x + product(a.view(t, self.nh * self.hd), "o")
            gate, up = product(self._rms(x, ly["ln2"]), "gate_up").chunk(2, -1)
            x = x + product(torch.nn.functional.silu(gate) * up, "down")
        last = torch.tensor([c - 1 for c in cu[1:]], dtype=torch.int64, device=dev)
        logits = torch.nn.functional.linear(self._rms(x[last], self.norm), self.head)
        self._commit(pages, lens)
        return logits
