"""Timed cases of the operators that take a chunk of new tokens through a decoder layer: the 8-bit integer product
with scales per token and channel (`ops.linear_w8`), the per-head norm + rotation + append to a paged cache
(`paged.norm_rope_append`) and the attention of the new tokens over that cache (`paged.attention`).

`run` computes each in its plain form from elementary torch operations in 32 bits, or, with `own`, through the
package. Layer sizes are those of the decoders the package is benchmarked on (hidden 1536, 2048, 3584; 12 to 28
query heads of 64 or 128 over 2 or 4 key heads).
"""
import math
import pathlib
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"
THETA, EPS = 1e6, 1e-6


# ------------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one decode step's token of one sequence: latency only
        dict(name="append_step_1", op="append", tokens=1, nh=16, nkv=2, hd=128, dtype="fp16", page=16, norm=False, at=700),
        # one step of a batch of sequences, small heads with norms
        dict(name="append_batch_61", op="append", tokens=61, nh=14, nkv=2, hd=64, dtype="bf16", page=32, norm=True, at=9000),
        # a long prompt's chunk
        dict(name="append_chunk_8192", op="append", tokens=8192, nh=28, nkv=4, hd=128, dtype="fp16", page=64, norm=True, at=24000),
        # a decode step of one sequence at a short context
        dict(name="attn_step_1", op="attention", seqs=1, new=1, context=700, nh=16, nkv=2, hd=128, dtype="fp16", page=16),
        # a decode step of a serving batch whose contexts differ
        dict(name="attn_step_96", op="attention", seqs=96, new=1, context=8192, nh=28, nkv=4, hd=128, dtype="bf16", page=64),
        # a follow-up prompt over a cached conversation, odd lengths
        dict(name="attn_chunk_509", op="attention", seqs=1, new=509, context=4093, nh=16, nkv=2, hd=128, dtype="fp16", page=32),
        # a mixed batch: single tokens, short and long chunks, ragged contexts
        dict(name="attn_ragged_12", op="attention", seqs=12, new=900, context=6000, nh=14, nkv=2, hd=64, dtype="bf16", page=16),
        # a chunk of a long document's prompt
        dict(name="attn_long_6000", op="attention", seqs=1, new=6000, context=32000, nh=28, nkv=4, hd=128, dtype="bf16", page=128),
        # a decode step's projection: the weight stream
        dict(name="w8_step_1", op="linear", rows=1, k=2048, n=11008, dtype="fp16", bias=False),
        # a batch's decode step: the fused q, k, v projection with its bias
        dict(name="w8_batch_33", op="linear", rows=33, k=3584, n=4608, dtype="bf16", bias=True),
        # a short prompt through the fused gate and up projection, an odd row count
        dict(name="w8_chunk_509", op="linear", rows=509, k=1536, n=17920, dtype="fp16", bias=False),
        # a long prompt's chunk through the down projection: the largest product
        dict(name="w8_prompt_8192", op="linear", rows=8192, k=18944, n=3584, dtype="bf16", bias=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "linear"))
    dtype = rng.choice(("fp16", "bf16"))
    nh, nkv, hd = rng.choice(((16, 2, 128), (28, 4, 128), (14, 2, 64), (12, 2, 128), (8, 8, 64)))
    page = rng.choice((16, 32, 48, 64, 128, 256))
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 8192), nh=nh, nkv=nkv, hd=hd, dtype=dtype, page=page,
                    norm=rng.random() < 0.5, at=_log(rng, 16, 24000))
    if op == "attention":
        if rng.random() < 0.4:
            seqs, new = _log(rng, 1, 128), 1
            context = _log(rng, 16, min(32000, 96 * 8192 // seqs))
        else:
            seqs = _log(rng, 1, 16)
            context = _log(rng, 128, 32000)
            new = _log(rng, 2, min(context, int(5e9 / (nh * seqs * context)), 6000))
        return dict(op=op, seqs=seqs, new=new, context=context, nh=nh, nkv=nkv, hd=hd, dtype=dtype, page=page)
    n = rng.choice((_log(rng, 128, 18944), 8 * _log(rng, 16, 2368)))
    k = rng.choice((_log(rng, 128, 18944), 128 * rng.randint(1, 148)))
    return dict(op=op, rows=_log(rng, 1, max(2, min(8192, int(5e11 / (n * k))))), k=k, n=n, dtype=dtype, bias=rng.random() < 0.5)


def _lengths(case):
    """(new tokens, context) of each sequence: the longest as the case says, the others spread below, some at 1."""
    rng = random.Random(case["seqs"] * 1000003 + case["new"] * 1009 + case["context"])
    new, ctx = [case["new"]], [case["context"]]
    for i in range(1, case["seqs"]):
        n = 1 if i % 3 == 1 else max(1, int(case["new"] * rng.random()))
        new.append(n)
        ctx.append(max(n, int(case["context"] * rng.random())))
    return new, ctx


# ----------------------------------------------------------------------------------------------------- the inputs

def _package():
    root = pathlib.Path(__file__).resolve().parent.parent / "lowbit-kernels_b200"
    if str(root) not in sys.path:
        sys.path.insert(0, str(root))
    from lowbit import ops, paged
    return ops, paged


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device=DEVICE, generator=gen) * std).to(dt)

    state = _PREPARE[case["op"]](case, gen, dt, normal)
    state["op"] = case["op"]
    if own:   # the handles a program keeps: the weight's and the cache's
        ops, paged = _package()
        state["lib"] = ops, paged
        if case["op"] == "linear":
            state["weight"] = ops.W8Weight(state["w"], state["w_scale"])
        else:
            state["cache"] = paged.PagedCache.from_tensors(state["k"], state["v"])
    return state


def _prepare_append(case, gen, dt, normal):
    t, nh, nkv, hd, page = (case[k] for k in ("tokens", "nh", "nkv", "hd", "page"))
    pages = (t + case["at"]) // page + 2
    order = torch.randperm(pages, device=DEVICE, generator=gen)
    pos = torch.arange(t, device=DEVICE) + case["at"]
    return dict(nh=nh, nkv=nkv, hd=hd, page=page, qkv=normal(t, (nh + 2 * nkv) * hd, std=1.5), pos=pos,
                slots=order[pos // page] * page + pos % page,
                q_norm=(1 + 0.1 * torch.randn(hd, device=DEVICE, generator=gen)).to(dt) if case["norm"] else None,
                k_norm=(1 + 0.1 * torch.randn(hd, device=DEVICE, generator=gen)).to(dt) if case["norm"] else None,
                inv_freq=1.0 / THETA ** (torch.arange(0, hd, 2, device=DEVICE, dtype=torch.float32) / hd),
                k=torch.zeros(pages, nkv, page, hd, device=DEVICE, dtype=dt),
                v=torch.zeros(pages, nkv, page, hd, device=DEVICE, dtype=dt))


def _prepare_attention(case, gen, dt, normal):
    nh, nkv, hd, page = (case[k] for k in ("nh", "nkv", "hd", "page"))
    new, ctx = _lengths(case)
    need = [-(-c // page) for c in ctx]
    width, pages = max(need), sum(need) + 1
    order = torch.randperm(pages, device=DEVICE, generator=gen).to(torch.int32)
    at = torch.tensor([0] + need, device=DEVICE).cumsum(0)
    col = torch.arange(width, device=DEVICE)
    table = torch.where(col < torch.tensor(need, device=DEVICE)[:, None], order[(at[:-1, None] + col).clamp(max=pages - 1)], 0)
    cu = torch.tensor([0] + new, device=DEVICE).cumsum(0).to(torch.int32)
    return dict(nh=nh, nkv=nkv, hd=hd, page=page, q=normal(sum(new), nh, hd, std=1.5), k=normal(pages, nkv, page, hd),
                v=normal(pages, nkv, page, hd), table=table.to(torch.int32).contiguous(),
                lens=torch.tensor(ctx, device=DEVICE, dtype=torch.int32), cu=cu, new=case["new"], context=case["context"])


def _prepare_linear(case, gen, dt, normal):
    m, k, n = case["rows"], case["k"], case["n"]
    x = normal(m, k)
    x[:, :: 97] *= 8   # activations have a few wide channels
    return dict(x=x, w=torch.randint(-127, 128, (n, k), device=DEVICE, dtype=torch.int8, generator=gen),
                w_scale=(0.5 + torch.rand(n, device=DEVICE, generator=gen)) * (0.06 / 127),
                bias=normal(n, std=0.2) if case["bias"] else None)


_PREPARE = dict(append=_prepare_append, attention=_prepare_attention, linear=_prepare_linear)


# ------------------------------------------------------------------------------------------------------- one pass

def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


def _own_append(s):
    q = s["lib"][1].norm_rope_append(s["qkv"], s["cache"], s["pos"], s["slots"], s["nh"], s["inv_freq"],
                                     q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
    return q, s["k"], s["v"]


def _own_attention(s):
    return s["lib"][1].attention(s["q"], s["cache"], s["table"], s["lens"], s["cu"], max_new=s["new"])


def _own_linear(s):
    return s["lib"][0].linear_w8(s["x"], s["weight"], bias=s["bias"])


def _rotate(x, pos, inv_freq):
    angle = pos.float()[:, None] * inv_freq
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_append(s):
    nh, nkv, hd, page = s["nh"], s["nkv"], s["hd"], s["page"]
    x = s["qkv"].float().view(-1, nh + 2 * nkv, hd)
    q, k, v = x.split((nh, nkv, nkv), 1)
    if s["q_norm"] is not None:
        q = q * (q.square().mean(-1, keepdim=True) + EPS).rsqrt() * s["q_norm"].float()
        k = k * (k.square().mean(-1, keepdim=True) + EPS).rsqrt() * s["k_norm"].float()
    q, k = _rotate(q, s["pos"], s["inv_freq"]), _rotate(k, s["pos"], s["inv_freq"])
    at, row = s["slots"] // page, s["slots"] % page
    s["k"][at, :, row] = k.to(s["k"].dtype)
    s["v"][at, :, row] = v.to(s["v"].dtype)
    return q.to(s["qkv"].dtype), s["k"], s["v"]


def _plain_attention(s):
    nh, nkv, hd, page, q, n = s["nh"], s["nkv"], s["hd"], s["page"], s["q"], s["new"]
    g, total, seqs = nh // nkv, q.shape[0], s["lens"].shape[0]
    j = torch.arange(s["context"], device=q.device)
    at = s["table"][:, j // page]
    k = s["k"][at, :, j % page].float().permute(0, 2, 3, 1)      # [seqs, nkv, hd, context]
    v = s["v"][at, :, j % page].float().permute(0, 2, 1, 3)
    i = torch.arange(n, device=q.device)
    t, count = s["cu"][:-1, None] + i, (s["cu"][1:] - s["cu"][:-1])[:, None]
    rows = q[t.clamp(max=total - 1)].float().view(seqs, n, nkv, g, hd).permute(0, 2, 3, 1, 4)
    score = torch.matmul(rows.reshape(seqs, nkv, g * n, hd), k).view(seqs, nkv, g, n, -1).mul_(1 / math.sqrt(hd))
    last = s["lens"][:, None] - count + i                        # the last key each new token sees
    score.masked_fill_((j > last[..., None])[:, None, None], float("-inf"))
    score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total_w = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(seqs, nkv, g * n, -1), v).view(seqs, nkv, g, n, hd) / total_w.clamp(min=1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs * n, nh, hd).to(q.dtype)
    return out[_unpad(s["cu"], n, total)]


def _unpad(cu, n, total):
    """The row of each token in the [sequence, n] padded order."""
    t = torch.arange(total, device=cu.device)
    seq = (t[:, None] >= cu[1:]).sum(1)
    return seq * n + t - cu[seq]


def _plain_linear(s):
    x = s["x"].float()
    amax = x.abs().amax(1, keepdim=True)
    q = (x * torch.where(amax > 0, torch.full_like(amax, 127.0) / amax, 0.0)).round()
    y = torch.matmul(q, s["w"].float().t()) * (amax / 127.0) * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


_OWN = dict(append=_own_append, attention=_own_attention, linear=_own_linear)
_PLAIN = dict(append=_plain_append, attention=_plain_attention, linear=_plain_linear)


# ----------------------------------------------------------------------------------------- what a pass has to do

def work(case):
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return dict(bytes=2 * m * k + n * k + 4 * n + 2 * m * n + 2 * n * case["bias"], flops=2 * m * n * k)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    if case["op"] == "append":
        t = case["tokens"]
        return dict(bytes=t * (2 * (nh + 2 * nkv) * hd * 2 + 16), flops=t * (nh + nkv) * hd * (7 if case["norm"] else 3))
    new, ctx = _lengths(case)
    seen = sum(n * c - n * (n - 1) // 2 for n, c in zip(new, ctx))
    return dict(bytes=4 * sum(new) * nh * hd + sum(ctx) * nkv * hd * 4, flops=4 * hd * nh * seen)


# -------------------------------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["op"]](s)


def _exact_append(s):
    nh, nkv, hd, page = s["nh"], s["nkv"], s["hd"], s["page"]
    x = s["qkv"].double().view(-1, nh + 2 * nkv, hd)
    angle = s["pos"].double()[:, None, None] * s["inv_freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle)

    def head(h, w):
        if w is not None:
            h = h / torch.sqrt((h * h).sum(-1, keepdim=True) / hd + EPS) * w.double()
        z = torch.complex(h[..., : hd // 2], h[..., hd // 2:]) * turn
        return torch.cat((z.real, z.imag), -1)

    k, v = s["k"].double(), s["v"].double()
    flat = s["slots"]
    for c, new in ((k, head(x[:, nh:nh + nkv], s["k_norm"])), (v, x[:, nh + nkv:])):
        for h in range(nkv):
            rows = c[:, h].reshape(-1, hd)
            rows[flat] = new[:, h]
            c[:, h] = rows.view(-1, page, hd)
    return head(x[:, :nh], s["q_norm"]), k, v


def _exact_attention(s):
    nh, nkv, hd, page = s["nh"], s["nkv"], s["hd"], s["page"]
    g, q = nh // nkv, s["q"].double()
    out = torch.zeros_like(q)
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    for i, length in enumerate(lens):
        a, b = cu[i], cu[i + 1]
        at = s["table"][i, : -(-length // page)].long()
        last = length - (b - a) + torch.arange(b - a, device=q.device)
        mask = torch.arange(length, device=q.device) > last[:, None]
        for h in range(nh):
            k = s["k"][at, h // g].reshape(-1, hd)[:length].double()
            v = s["v"][at, h // g].reshape(-1, hd)[:length].double()
            score = (q[a:b, h] @ k.t()) / math.sqrt(hd)
            out[a:b, h] = torch.softmax(score.masked_fill(mask, float("-inf")), -1) @ v
    return out


def _exact_linear(s):
    x = s["x"].double()
    amax = x.abs().amax(1, keepdim=True)
    q = torch.where(amax > 0, torch.round(x * 127 / amax), torch.zeros_like(x))
    y = (q @ s["w"].double().t()) * (amax / 127) * s["w_scale"].double()
    return y if s["bias"] is None else y + s["bias"].double()


_EXACT = dict(append=_exact_append, attention=_exact_attention, linear=_exact_linear)
