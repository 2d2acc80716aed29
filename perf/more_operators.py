"""Timed cases of the operators that take a step of drafted tokens through a decoder over the paged cache: page tables,
slots, positions and tree masks built on the GPU from the request lengths (`paged.plan`), the attention of a tree of
drafted tokens over the cache (`paged.tree_attention`), the acceptance of the drafts (`paged.verify`), the move of the
accepted tokens' K and V rows to where they belong (`paged.compact`), and the product in 8-bit floating point with a scale
for each block of 128 (`ops.linear_f8`).

`run` computes each in its plain form from elementary torch operations in 32 bits, or, with `own`, through the
package. Layer sizes are those of the decoders the package is benchmarked on.
"""
import math
import pathlib
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"
BLOCK = 128                # of the 8-bit products' scales
LEAST = 2.0 ** -100        # the least maximum of a block of activations


# ------------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # a small serving batch, each sequence with a tree of drafted tokens: latency only
        dict(name="plan_trees_16", op="plan", seqs=16, new=31, context=4000, page=16, tree=True),
        # prompts of a large batch in one call: tens of thousands of tokens
        dict(name="plan_prompts_48", op="plan", seqs=48, new=2048, context=6000, page=64, tree=False),
        # one sequence's first drafts at a short context
        dict(name="tree_8", op="tree", seqs=1, new=8, context=700, nh=16, nkv=2, hd=128, dtype="fp16", page=16),
        # a serving batch with trees of different sizes over contexts of different lengths
        dict(name="tree_batch_32", op="tree", seqs=32, new=25, context=8192, nh=28, nkv=4, hd=128, dtype="bf16", page=64),
        # a wide tree over a long document
        dict(name="tree_long_255", op="tree", seqs=1, new=255, context=32000, nh=28, nkv=4, hd=128, dtype="bf16", page=128),
        # one sequence's drafts against the whole vocabulary
        dict(name="verify_8", op="verify", seqs=1, new=8, vocab=151936, dtype="fp16"),
        # a serving batch's
        dict(name="verify_batch_64", op="verify", seqs=64, new=31, vocab=152064, dtype="bf16"),
        # one sequence's accepted drafts in all layers
        dict(name="compact_1", op="compact", seqs=1, new=25, context=700, layers=36, nkv=2, hd=128, dtype="fp16", page=16),
        # a serving batch's
        dict(name="compact_64", op="compact", seqs=64, new=61, context=300, layers=28, nkv=4, hd=128, dtype="bf16", page=64),
        # a decode step's projection: the weight stream
        dict(name="f8_step_1", op="linear", rows=1, k=2048, n=11008, dtype="fp16", bias=False),
        # a tree's tokens through the fused q, k, v projection with its bias
        dict(name="f8_tree_61", op="linear", rows=61, k=3584, n=4608, dtype="bf16", bias=True),
        # a long prompt's chunk through the down projection: the largest product
        dict(name="f8_prompt_8192", op="linear", rows=8192, k=18944, n=3584, dtype="bf16", bias=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("plan", "tree", "tree", "verify", "compact", "linear", "linear"))
    dtype = rng.choice(("fp16", "bf16"))
    nh, nkv, hd = rng.choice(((16, 2, 128), (28, 4, 128), (14, 2, 64), (12, 2, 128), (8, 8, 64)))
    page = rng.choice((16, 32, 48, 64, 128, 256))
    if op == "plan":
        tree, seqs = rng.random() < 0.5, _log(rng, 1, 512)
        new = _log(rng, 1, 128) if tree else _log(rng, 1, min(2048, 98304 // seqs))
        return dict(op=op, seqs=seqs, new=new, context=_log(rng, 16, 8000), page=page, tree=tree)
    if op == "tree":
        seqs, new = _log(rng, 1, 64), _log(rng, 1, 255)
        most = min(32000, int(2.2e8 / (nh * seqs * new)), 300000 // seqs)
        return dict(op=op, seqs=seqs, new=new, context=new + _log(rng, 16, max(17, most)), nh=nh, nkv=nkv, hd=hd, dtype=dtype,
                    page=page)
    if op == "verify":
        seqs = _log(rng, 1, 64)
        vocab = rng.choice((151936, 152064, _log(rng, 1000, 152064)))
        return dict(op=op, seqs=seqs, new=_log(rng, 1, min(255, 2000 // seqs)), vocab=vocab, dtype=dtype)
    if op == "compact":
        return dict(op=op, seqs=_log(rng, 1, 64), new=_log(rng, 8, 128), context=_log(rng, 130, 300),
                    layers=rng.randint(1, 28), nkv=nkv if nkv < 8 else 2, hd=hd, dtype=dtype, page=page)
    n = rng.choice((_log(rng, 128, 18944), 128 * rng.randint(1, 148)))
    k = rng.choice((_log(rng, 128, 18944), 128 * rng.randint(1, 148)))
    return dict(op=op, rows=_log(rng, 1, max(2, min(8192, int(5e11 / (n * k))))), k=k, n=n, dtype=dtype, bias=rng.random() < 0.5)


def _lengths(case):
    """(new tokens, context) of each sequence: the longest as the case says, the others spread below, some at 1 new."""
    rng = random.Random(case["seqs"] * 1000003 + case["new"] * 1009 + case.get("context", 0))
    context = case.get("context", case["new"])
    new, ctx = [case["new"]], [max(case["new"], context)]
    for i in range(1, case["seqs"]):
        n = 1 if i % 7 == 3 else max(1, int(case["new"] * (0.2 + 0.8 * rng.random())))
        new.append(n)
        ctx.append(n + int((ctx[0] - case["new"]) * rng.random()))
    return new, ctx


def _parents(rng, n):
    """A tree of n drafted tokens, token 0 its root: each token's parent, earlier than itself."""
    return [-1] + [rng.randint(max(0, i - 1 - i // 2), i - 1) for i in range(1, n)]


def _ancestors(parents, words):
    """Each token's row of bits: its ancestors and itself."""
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    return [[((r >> 32 * w) & 0xFFFFFFFF) - (1 << 32 if r >> (32 * w + 31) & 1 else 0) for w in range(words)] for r in rows]


# ----------------------------------------------------------------------------------------------------- the inputs

def _package():
    root = pathlib.Path(__file__).resolve().parent.parent / "lowbit-kernels_b200"
    if str(root) not in sys.path:
        sys.path.insert(0, str(root))
    from lowbit import ops, paged
    return ops, paged


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = _PREPARE[case["op"]](case, gen, random.Random(seed), DTYPES[case.get("dtype", "fp16")])
    state["op"] = case["op"]
    if own:   # the handles a program keeps: the weight's and the caches'
        ops, paged = _package()
        state["lib"] = ops, paged
        if case["op"] == "linear":
            state["weight"] = ops.F8Weight(state["w"], state["w_scale"])
        elif case["op"] == "tree":
            state["cache"] = paged.PagedCache.from_tensors(state["k"], state["v"])
        elif case["op"] == "compact":
            state["caches"] = [paged.PagedCache.from_tensors(k, v) for k, v in zip(state["k"], state["v"])]
    return state


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEVICE)


def _cu(new):
    return _ints([0] + new).cumsum(0).to(torch.int32)


def _table(gen, counts, width, pages):
    """A page table whose rows hold that many pages each, in no order; zeros behind them."""
    order = torch.randperm(pages, device=DEVICE, generator=gen).to(torch.int32)
    at = _ints([0] + counts).cumsum(0)
    col = torch.arange(width, device=DEVICE)
    table = torch.where(col < _ints(counts)[:, None], order[(at[:-1, None] + col).clamp(max=pages - 1)], 0)
    return table.to(torch.int32).contiguous(), order[sum(counts):].contiguous()


def _prepare_plan(case, gen, rng, dt):
    page, (new, ctx) = case["page"], _lengths(case)
    lens = [c - n for n, c in zip(new, ctx)]
    held = [-(-v // page) for v in lens]
    width = max(-(-c // page) for c in ctx)
    table, free = _table(gen, held, width, sum(-(-c // page) for c in ctx) + 5)
    parents = [p for n in new for p in _parents(rng, n)] if case["tree"] else None
    return dict(page=page, new=case["new"], total=sum(new), table=table, lens=_ints(lens), new_lens=_ints(new), held=_ints(held),
                free=free, count=_ints([free.numel()]), parents=None if parents is None else _ints(parents))


def _prepare_tree(case, gen, rng, dt):
    nh, nkv, hd, page = (case[k] for k in ("nh", "nkv", "hd", "page"))
    new, ctx = _lengths(case)
    need = [-(-c // page) for c in ctx]
    table, _ = _table(gen, need, max(need), sum(need) + 1)
    words = -(-case["new"] // 32)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device=DEVICE, generator=gen) * std).to(dt)

    return dict(nh=nh, nkv=nkv, hd=hd, page=page, new=case["new"], context=max(ctx), q=normal(sum(new), nh, hd, std=1.5),
                k=normal(sum(need) + 1, nkv, page, hd), v=normal(sum(need) + 1, nkv, page, hd), table=table, lens=_ints(ctx),
                cu=_cu(new), mask=_ints([row for n in new for row in _ancestors(_parents(rng, n), words)]))


def _prepare_verify(case, gen, rng, dt):
    new, vocab = _lengths(case)[0], case["vocab"]
    total = sum(new)
    logits = (torch.randn(total, vocab, device=DEVICE, generator=gen) * 2).to(dt)
    # most rows have one likely token, which a drafted child often is; some have only what chance made largest
    likely = torch.randint(0, vocab, (total,), device=DEVICE, generator=gen)
    rows = [i for i in range(total) if rng.random() < 0.85]
    logits[_ints(rows, torch.int64), likely[_ints(rows, torch.int64)]] = 20.0
    likely, tokens, parents, at = likely.tolist(), [], [], 0
    for n in new:
        tree = _parents(rng, n)
        tokens += [likely[at + p] if p >= 0 and rng.random() < 0.6 else rng.randrange(vocab) for p in tree]
        parents += tree
        at += n
    return dict(logits=logits, tokens=_ints(tokens, torch.int64), parents=_ints(parents), cu=_cu(new), new=case["new"], seqs=len(new))


def _prepare_compact(case, gen, rng, dt):
    nkv, hd, page, layers = (case[k] for k in ("nkv", "hd", "page", "layers"))
    new, ctx = _lengths(case)
    need = [-(-c // page) for c in ctx]
    table, _ = _table(gen, need, max(need), sum(need) + 1)
    # paths of up to seven tokens, one of each level of the tree; a moved token comes from behind the path, as in a tree
    # whose first level is as wide, so that a second pass moves the same rows
    longest, paths, counts = 7, [], []
    for n in new:
        path, length = [0], min(longest, 1 + n // 8)
        for d in range(1, length):
            path.append(d if path == list(range(d)) and rng.random() < 0.4 else rng.randint(max(longest, path[-1] + 1), n - length + d))
        counts.append(len(path))
        paths.append(path + [-1] * (longest - len(path)))
    shape = (layers, sum(need) + 1, nkv, page, hd)
    return dict(page=page, k=torch.randn(shape, device=DEVICE, generator=gen, dtype=dt),
                v=torch.randn(shape, device=DEVICE, generator=gen, dtype=dt), table=table, lens=_ints(ctx), cu=_cu(new),
                path=_ints(paths), accepted=_ints(counts))


def _prepare_linear(case, gen, rng, dt):
    m, k, n = case["rows"], case["k"], case["n"]
    x = torch.randn(m, k, device=DEVICE, generator=gen)
    x[:, :: 97] *= 8   # activations have a few wide channels
    w = (torch.randn(n, k, device=DEVICE, generator=gen) * 110).clamp_(-448, 448).to(torch.float8_e4m3fn)
    blocks = torch.rand(-(-n // BLOCK), -(-k // BLOCK), device=DEVICE, generator=gen)
    return dict(x=x.to(dt), w=w, w_scale=(0.5 + blocks) * (0.02 / 110),
                bias=(torch.randn(n, device=DEVICE, generator=gen) * 0.2).to(dt) if case["bias"] else None)


_PREPARE = dict(plan=_prepare_plan, tree=_prepare_tree, verify=_prepare_verify, compact=_prepare_compact, linear=_prepare_linear)


# ------------------------------------------------------------------------------------------------------- one pass

def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


def _own_plan(s):
    p = s["lib"][1].plan(s["table"], s["lens"], s["new_lens"], s["page"], s["total"], held=s["held"], free_pages=s["free"],
                         free_count=s["count"], parents=s["parents"], max_new=s["new"])
    return s["table"], p.cu_new, p.seq_lens, p.positions, p.slots, p.held, p.free_count, p.mask


def _own_tree(s):
    return s["lib"][1].tree_attention(s["q"], s["cache"], s["table"], s["lens"], s["cu"], s["mask"], max_new=s["new"])


def _own_verify(s):
    v = s["lib"][1].verify(s["logits"], s["tokens"], s["parents"], s["cu"], max_new=s["new"])
    return v.accepted, v.path, v.next, v.targets


def _own_compact(s):
    lens = s["lib"][1].compact(s["caches"], s["table"], s["lens"], s["cu"], s["path"], s["accepted"])
    return lens, s["k"], s["v"]


def _own_linear(s):
    return s["lib"][0].linear_f8(s["x"], s["weight"], bias=s["bias"])


def _places(cu, total):
    """Each token's sequence, and its place in it."""
    t = torch.arange(total, device=cu.device)
    seq = (t[:, None] >= cu[1:]).sum(1)
    return seq, t - cu[seq]


def _plain_plan(s):
    page, table, lens, new, total = s["page"], s["table"], s["lens"], s["new_lens"], s["total"]
    cu = torch.cat((torch.zeros_like(new[:1]), new.cumsum(0).to(torch.int32)))
    after = lens + new
    need = ((after + page - 1) // page - s["held"]).clamp(min=0)
    ends = need.cumsum(0)
    fits = (need == 0) | (ends <= s["count"])
    need = torch.where(fits, need, 0)
    col = torch.arange(table.shape[1], device=table.device) - s["held"][:, None]      # of the pages taken
    at = s["count"] - 1 - ((ends - need)[:, None] + col)
    table.copy_(torch.where((col >= 0) & (col < need[:, None]), s["free"][at.clamp(0, s["free"].numel() - 1)], table))
    seq, i = _places(cu, total)
    key = lens[seq] + i
    slots = table[seq, (key // page).clamp(max=table.shape[1] - 1)].long() * page + key % page
    mask, depth = None, i
    if s["parents"] is not None:
        n = s["new"]
        see = torch.zeros(lens.shape[0], n, n, device=table.device)                   # by one step, or none
        see[seq, i, i] = 1.0
        see[seq, i, torch.where(s["parents"] >= 0, s["parents"].long(), i)] = 1.0
        for _ in range(max(1, (n - 1).bit_length())):
            see = torch.matmul(see, see).clamp(max=1.0)
        seen = see[seq, i] > 0.5
        depth = seen.sum(1) - 1
        words = -(-n // 32)
        seen = torch.nn.functional.pad(seen, (0, 32 * words - n)).view(total, words, 32).long()
        mask = (seen << torch.arange(32, device=table.device)).sum(-1)
        mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32)
    return (table, cu, torch.where(fits, after, 0), (lens[seq] + depth).long(), torch.where(fits[seq], slots, -1),
            s["held"] + need, (s["count"] - need.sum()).to(torch.int32), mask)


def _plain_tree(s):
    nh, nkv, hd, page, q, n = s["nh"], s["nkv"], s["hd"], s["page"], s["q"], s["new"]
    g, total, seqs = nh // nkv, q.shape[0], s["lens"].shape[0]
    j = torch.arange(s["context"], device=q.device)
    at = s["table"][:, j // page]
    k = s["k"][at, :, j % page].float().permute(0, 2, 3, 1)      # [seqs, nkv, hd, context]
    v = s["v"][at, :, j % page].float().permute(0, 2, 1, 3)
    i = torch.arange(n, device=q.device)
    t, count = (s["cu"][:-1, None] + i).clamp(max=total - 1), (s["cu"][1:] - s["cu"][:-1])[:, None]
    rows = q[t].float().view(seqs, n, nkv, g, hd).permute(0, 2, 3, 1, 4)
    score = torch.matmul(rows.reshape(seqs, nkv, g * n, hd), k).view(seqs, nkv, g, n, -1).mul_(1 / math.sqrt(hd))
    drafted = j - (s["lens"][:, None] - count)                   # the key's place among the new tokens
    bit = drafted.clamp(0, n - 1)
    word = s["mask"][t][:, :, :].gather(2, (bit // 32)[:, None].expand(seqs, n, -1))
    sees = (drafted < 0)[:, None] | (((word >> (bit % 32)[:, None]) & 1).bool() & (drafted < count)[:, None])
    score.masked_fill_(~sees[:, None, None], float("-inf"))
    score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total_w = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(seqs, nkv, g * n, -1), v).view(seqs, nkv, g, n, hd) / total_w.clamp(min=1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs * n, nh, hd).to(q.dtype)
    seq, i = _places(s["cu"], total)
    return out[seq * n + i]


def _plain_verify(s):
    logits, tokens, parents, cu, n = s["logits"], s["tokens"], s["parents"], s["cu"], s["new"]
    targets = logits.float().argmax(-1)
    i = torch.arange(n, device=cu.device)
    count = (cu[1:] - cu[:-1])[:, None]
    t = (cu[:-1, None] + i).clamp(max=tokens.shape[0] - 1).long()
    token, parent, target = tokens[t], parents[t], targets[t]
    cur = torch.zeros_like(count[:, 0]).long()
    path, accepted, alive = [cur], torch.ones_like(count[:, 0]), torch.ones_like(cur, dtype=torch.bool)
    for _ in range(1, n):
        child = (parent == cur[:, None]) & (token == target.gather(1, cur[:, None])) & (i < count)
        child = torch.where(child, i, n).amin(1)
        alive = alive & (child < n)
        cur = torch.where(alive, child, cur)
        accepted = accepted + alive
        path.append(torch.where(alive, child, -1))
    return accepted.to(torch.int32), torch.stack(path, 1).to(torch.int32), target.gather(1, cur[:, None])[:, 0], targets


def _plain_compact(s):
    page, table, path, accepted = s["page"], s["table"], s["path"], s["accepted"]
    start = s["lens"] - (s["cu"][1:] - s["cu"][:-1])
    d = torch.arange(path.shape[1], device=path.device)
    # (a row that is not moved is written over itself)
    src = (start[:, None] + torch.where(d < accepted[:, None], path, 0)).long()
    dst = (start[:, None] + torch.where(d < accepted[:, None], d, 0)).long()
    seq = torch.arange(path.shape[0], device=path.device)[:, None]
    for c in (s["k"], s["v"]):
        rows = c[:, table[seq, src // page].long(), :, src % page]
        c[:, table[seq, dst // page].long(), :, dst % page] = rows
    return start + accepted, s["k"], s["v"]


def _groups(x):
    """x [M, K] as [M, blocks of K, 128], zeros behind K."""
    k = x.shape[1]
    return torch.nn.functional.pad(x, (0, -k % BLOCK)).view(x.shape[0], -1, BLOCK)


def _plain_linear(s):
    x, k = _groups(s["x"].float()), s["x"].shape[1]
    amax = x.abs().amax(2, keepdim=True).clamp(min=LEAST)
    q = (x * (torch.full_like(amax, 448.0) / amax)).to(torch.float8_e4m3fn).float()
    x = (q * (amax / torch.full_like(amax, 448.0))).view(x.shape[0], -1)[:, :k]
    n = s["w"].shape[0]
    w = s["w"].float() * s["w_scale"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = torch.matmul(x, w.t())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


_OWN = dict(plan=_own_plan, tree=_own_tree, verify=_own_verify, compact=_own_compact, linear=_own_linear)
_PLAIN = dict(plan=_plain_plan, tree=_plain_tree, verify=_plain_verify, compact=_plain_compact, linear=_plain_linear)


# ----------------------------------------------------------------------------------------- what a pass has to do

def work(case):
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return dict(bytes=2 * m * k + n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK) + 2 * m * n + 2 * n * case["bias"], flops=2 * m * n * k)
    new, ctx = _lengths(case)
    if case["op"] == "plan":
        page = case["page"]
        pages = sum(-(-c // page) - -(-(c - n) // page) for n, c in zip(new, ctx))
        row = 16 + case["tree"] * (4 + 4 * -(-case["new"] // 32))
        return dict(bytes=24 * len(new) + 8 * pages + row * sum(new), flops=4 * sum(new))
    if case["op"] == "verify":
        return dict(bytes=2 * sum(new) * case["vocab"] + 20 * sum(new), flops=sum(new) * case["vocab"])
    if case["op"] == "compact":   # (the rows that move on average)
        moved = sum(sum(1 - 0.4 ** d for d in range(1, min(7, 1 + n // 8))) for n in new)
        return dict(bytes=moved * case["layers"] * 2 * case["nkv"] * case["hd"] * 2 * 2 + 12 * len(new), flops=1)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    seen = sum(n * (c - n) + n * min(n, 2 * n.bit_length()) for n, c in zip(new, ctx))
    return dict(bytes=4 * sum(new) * nh * hd + sum(ctx) * nkv * hd * 4 + 4 * sum(new) * -(-case["new"] // 32), flops=4 * hd * nh * seen)


# -------------------------------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))


def _exact_plan(s):
    page, total = s["page"], s["total"]
    table, lens, new, held, free = (s[k].tolist() for k in ("table", "lens", "new_lens", "held", "free"))
    left = s["count"].item()
    parents = None if s["parents"] is None else s["parents"].tolist()
    cu, after, pos, slots, mask = [0], [], [], [], []
    for a, n in enumerate(new):
        for j in range(held[a], -(-(lens[a] + n) // page)):
            left -= 1
            table[a][j] = free[left]
            held[a] = j + 1
        tree = None if parents is None else parents[cu[-1]:cu[-1] + n]
        depth = []
        for i in range(n):
            at = lens[a] + i
            slots.append(table[a][at // page] * page + at % page)
            depth.append(i if tree is None else 0 if tree[i] < 0 else depth[tree[i]] + 1)
            pos.append(lens[a] + depth[-1])
        if tree is not None:
            mask += _ancestors(tree, -(-s["new"] // 32))
        cu.append(cu[-1] + n)
        after.append(lens[a] + n)
    assert len(slots) == total
    return (_ints(table), _ints(cu), _ints(after), _ints(pos, torch.int64), _ints(slots, torch.int64), _ints(held), _ints([left]),
            None if parents is None else _ints(mask))


def _exact_tree(s):
    nh, nkv, hd = s["nh"], s["nkv"], s["hd"]
    g, q = nh // nkv, s["q"].double()
    out = torch.zeros_like(q)
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    for a, length in enumerate(lens):
        t0, t1 = cu[a], cu[a + 1]
        n = t1 - t0
        at = s["table"][a, : -(-length // s["page"])].long()
        bits = torch.stack([s["mask"][t0:t1, b // 32] >> b % 32 & 1 for b in range(n)], 1).bool()
        hidden = torch.cat((torch.zeros(n, length - n, dtype=torch.bool, device=q.device), ~bits), 1)
        for h in range(nkv):
            k = s["k"][at, h].reshape(-1, hd)[:length].double()
            v = s["v"][at, h].reshape(-1, hd)[:length].double()
            score = torch.einsum("ngd,kd->gnk", q[t0:t1, h * g:(h + 1) * g], k) / math.sqrt(hd)
            p = torch.softmax(score.masked_fill(hidden, float("-inf")), -1)
            out[t0:t1, h * g:(h + 1) * g] = torch.einsum("gnk,kd->ngd", p, v)
    return out


def _exact_verify(s):
    best = []
    for row in s["logits"].split(64):
        row = row.double()
        best.append((row == row.amax(1, keepdim=True)).to(torch.uint8).argmax(1))
    targets = torch.cat(best)
    best, tokens, parents, cu, n = targets.tolist(), s["tokens"].tolist(), s["parents"].tolist(), s["cu"].tolist(), s["new"]
    accepted, paths, after = [], [], []
    for a, b in zip(cu, cu[1:]):
        path = [0]
        while True:
            child = [c for c in range(path[-1] + 1, b - a) if parents[a + c] == path[-1] and tokens[a + c] == best[a + path[-1]]]
            if not child:
                break
            path.append(child[0])
        accepted.append(len(path))
        after.append(best[a + path[-1]])
        paths.append(path + [-1] * (n - len(path)))
    return _ints(accepted), _ints(paths), _ints(after, torch.int64), targets


def _exact_compact(s):
    page, cu, lens = s["page"], s["cu"].tolist(), s["lens"].tolist()
    table, path, accepted = s["table"].tolist(), s["path"].tolist(), s["accepted"].tolist()
    src, dst, after = [], [], []
    for a, length in enumerate(lens):
        start = length - (cu[a + 1] - cu[a])
        for d in range(accepted[a]):
            for at, to in ((start + path[a][d], src), (start + d, dst)):
                to.append(table[a][at // page] * page + at % page)
        after.append(start + accepted[a])
    out = []
    for c in (s["k"], s["v"]):
        layers, pages, nkv, _, hd = c.shape
        flat = c.double().transpose(2, 3).reshape(layers, pages * page, nkv, hd)
        flat[:, _ints(dst, torch.int64)] = flat[:, _ints(src, torch.int64)]
        out.append(flat.view(layers, pages, page, nkv, hd).transpose(2, 3))
    return (_ints(after), *out)


def _exact_linear(s):
    k, n = s["x"].shape[1], s["w"].shape[0]
    y = torch.zeros(s["x"].shape[0], n, device=DEVICE, dtype=torch.float64)
    rows = torch.arange(n, device=DEVICE) // BLOCK
    for b, a in enumerate(range(0, k, BLOCK)):
        x = s["x"][:, a:a + BLOCK].double()
        amax = x.abs().amax(1, keepdim=True).clamp(min=LEAST)
        # the operator's own step to 8 bits is one product in 32 bits, which decides where a value between two steps goes
        up = x.float() * (torch.full_like(amax, 448.0, dtype=torch.float32) / amax.float())
        y += (up.to(torch.float8_e4m3fn).double() @ s["w"][:, a:a + BLOCK].double().t()) * (amax / 448) * s["w_scale"][rows, b].double()
    return y if s["bias"] is None else y + s["bias"].double()


_EXACT = dict(plan=_exact_plan, tree=_exact_tree, verify=_exact_verify, compact=_exact_compact, linear=_exact_linear)
