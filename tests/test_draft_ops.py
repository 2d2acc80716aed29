"""The operators of a step of drafted tokens against plain implementations, in 64 bits where they compute (B200 only, but for
the refusals of the C ABI, which come before any CUDA call).

Tolerances, with u = 2^-11 (fp16) or 2^-8 (bf16) the relative rounding of one stored value:
  * tree_attention: those of attention (test_chunk_ops.py), which differs in what a row sees alone;
  * linear_f8: the quantized activations are reproduced bit for bit (one fp32 quotient, product and rounding to e4m3).
    A block's 128 products, exact in fp32, are added by the tensor core 32 at a time: a step keeps at least fp32's 24 bits
    of the largest magnitude in it, so its up to 33 terms lose at most 33 * 2^-23 of that, and the four steps 2^-15.9 of
    A_b = sum |q w|. The scales' product and its multiply-add into the running sum: 3 * 2^-24 of A_b s t and 2^-24 of the sum a
    block. With A the sum of all s t A_b: u |y| + (2^-15.9 + (blocks + 3) 2^-24) (A + |bias|).
    On integers, with scales that are powers of two, nothing is rounded before the result: the test of exact sums allows u |y|.
  * plan, verify and compact compute whole numbers or move rows: equal.
Every tolerance adds 2^-24, half of fp16's smallest step, twice.
"""
import copy
import ctypes
import math
import pickle
import random
import re
import threading

import pytest
import torch

from lowbit import _lib
from test_chunk_ops import A, DTYPES, MIS, U, build, close, gen, message, mods, randn

gpu = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def status():
    return mods()[0].ext().lib.lb_device_error()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def i64(v):
    return torch.tensor(v, dtype=torch.int64, device="cuda")


def cu_of(new):
    return i32([0] + new).cumsum(0).to(torch.int32)


def tree(rng, n):
    return [-1] + [rng.randint(max(0, i - 9), i - 1) for i in range(1, n)] if n else []


def ancestors(parents):
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if 0 <= p < i else 0) | 1 << i)
    return rows


def words_of(rows, words):
    """Rows of bits (whole numbers) as int32 words."""
    out = [[(r >> 32 * w) & 0xFFFFFFFF for w in range(words)] for r in rows]
    return i32([[v - (1 << 32) if v >> 31 else v for v in r] for r in out]).view(len(rows), words)


# ----------------------------------------------------------------------------------------------------------- plan

def plain_plan(table, lens, new, page, tokens, held=None, free=None, count=0, parents=None, words=0):
    """The same in Python: what `plan` returns, and the table."""
    table, width = copy.deepcopy(table), len(table[0])
    cu, after, pos, slots, mask, held = [0], [], [], [], [], list(held) if held else None
    left, short = max(0, min(count, len(free or []))), False
    for s, (c, n) in enumerate(zip(lens, new)):
        c, n = max(0, c), max(0, n)
        start = cu[-1]
        served = start + n <= tokens and c + n <= width * page
        if held is not None and served:
            need = max(0, -(-(c + n) // page) - max(0, held[s]))
            if need and (short or need > left):
                served, short = False, True
            elif need:
                for j in range(need):
                    left -= 1
                    table[s][max(0, held[s]) + j] = free[left]
                held[s] = max(0, held[s]) + need
        if held is not None:
            held[s] = max(0, held[s])
        cu.append(min(tokens, start + n))
        after.append(c + n if served else 0)
        depth = []
        for i in range(cu[-1] - start):
            p = i - 1 if parents is None else parents[start + i]
            depth.append(depth[p] + 1 if 0 <= p < i else 0)
            pos.append(c + depth[-1])
            at = table[s][(c + i) // page] if served else -1
            slots.append(at * page + (c + i) % page if at >= 0 else -1)
        if parents is not None:
            mask += ancestors(parents[start:cu[-1]])
    spare = tokens - cu[-1]
    return dict(cu_new=cu, seq_lens=after, positions=pos + [0] * spare, slots=slots + [-1] * spare, held=held,
                free_count=[left] if held is not None else None,
                mask=None if parents is None else words_of(mask + [0] * spare, words)), table


def check_plan(got, want, table, want_table):
    for name, v in want.items():
        g = getattr(got, name)
        assert (g is None) == (v is None), name
        if v is not None:
            v = v if isinstance(v, torch.Tensor) else torch.tensor(v, dtype=g.dtype, device="cuda").view(g.shape)
            assert torch.equal(g, v), name
    assert table.tolist() == want_table


def plan_case(rng, seqs, most, page, shape, spare_tokens=0, spare_pages=3):
    new = [rng.choice((0, 1, rng.randint(0, most))) for _ in range(seqs)]
    lens = [rng.choice((0, page - 1, page, rng.randint(0, 6 * page))) for _ in range(seqs)]
    held = [-(-c // page) + rng.choice((0, 0, 2)) for c in lens]
    width = max(max(-(-(c + n) // page), h) for c, n, h in zip(lens, new, held)) + 1
    need = sum(max(0, -(-(c + n) // page) - h) for c, n, h in zip(lens, new, held))
    pages = list(range(sum(held) + need + spare_pages))
    rng.shuffle(pages)
    table, at = [], 0
    for h in held:
        table.append(pages[at:at + h] + [-5] * (width - h))
        at += h
    free = pages[at:]
    tokens = sum(new) + spare_tokens
    parents = [rng.choice((p, p, p, -1, 2000, i)) if shape == "odd" else p for n in new for i, p in enumerate(tree(rng, n))]
    return dict(table=table, lens=lens, new=new, held=held, free=free, tokens=tokens, page=page,
                parents=parents + [7] * spare_tokens if shape else None, most=max(new + [1]))


def run_plan(c, paging=True, count=None, out=None, table=None):
    _, paged = mods()
    t = i32(c["table"]) if table is None else table
    count = len(c["free"]) if count is None else count
    kw = dict(held=i32(c["held"]), free_pages=i32(c["free"]), free_count=i32([count])) if paging else {}
    if c["parents"] is not None:
        kw.update(parents=i32(c["parents"]), max_new=c["most"])
    got = paged.plan(t, i32(c["lens"]), i32(c["new"]), c["page"], c["tokens"], out=out, **kw)
    want, want_table = plain_plan(c["table"], c["lens"], c["new"], c["page"], c["tokens"], c["held"] if paging else None,
                                  c["free"] if paging else None, count, c["parents"], -(-c["most"] // 32))
    check_plan(got, want, t, want_table)
    return got


@gpu
@pytest.mark.parametrize("shape", [None, "tree", "odd"])
@pytest.mark.parametrize("seqs,most,page", [(1, 1, 16), (1, 70, 16), (3, 9, 48), (33, 61, 16), (64, 300, 64), (200, 40, 32),
                                            (1025, 3, 16), (1500, 33, 128), (8192, 2, 16)])
def test_plan(shape, seqs, most, page):
    rng = random.Random(seqs * 7 + most)
    for spare in (0, 13):
        run_plan(plan_case(rng, seqs, most, page, shape, spare_tokens=spare))
    c = plan_case(rng, seqs, most, page, shape)
    for s, (a, n) in enumerate(zip(c["lens"], c["new"])):   # a table that is complete as it is
        for j in range(-(-(a + n) // page)):
            c["table"][s][j] = rng.choice((rng.randint(0, 10 ** 6), (2 ** 31 - 1) // page))
    run_plan(c, paging=False)


@gpu
def test_plan_long_chains_and_trees_of_1024_tokens():
    rng = random.Random(4)
    for shape in ("chain", "tree", "star"):
        n = [1024, 1000, 5, 1024]
        c = dict(table=[[-1] * 70 for _ in n], lens=[0, 37, 2, 16], new=n, held=[0, 0, 0, 0], free=list(range(400)), page=16,
                 tokens=sum(n), most=1024)
        c["held"] = [0, 3, 1, 1]
        for s, h in enumerate(c["held"]):
            c["table"][s][:h] = [500 + 10 * s + j for j in range(h)]
        c["parents"] = [p for m in n for p in ([i - 1 for i in range(m)] if shape == "chain" else
                                               [-1] + [0] * (m - 1) if shape == "star" else tree(rng, m))]
        run_plan(c)


@gpu
def test_plan_refuses_sequences_that_do_not_fit():
    """Too few free pages, rows or table columns: the sequence is refused, those that need nothing are served."""
    rng = random.Random(11)
    for shape in (None, "tree"):
        c = plan_case(rng, 40, 50, 16, shape)
        for count in (0, 1, 5, len(c["free"]) // 2, len(c["free"]), len(c["free"]) + 50, -3):
            run_plan(c, count=count)
        for fewer in (1, c["tokens"] // 2, c["tokens"] - 1, c["tokens"]):
            d = dict(c, tokens=c["tokens"] - fewer)
            if shape:
                d["parents"] = c["parents"][:d["tokens"]]
            run_plan(d)
        d = copy.deepcopy(c)
        d["lens"][3], d["lens"][7], d["new"][5], d["new"][6] = 16 * len(c["table"][0]), 2 ** 31 - 1, -4, 0
        d["tokens"] = sum(max(0, n) for n in d["new"])
        if shape:
            d["parents"] = [p for n in d["new"] for p in tree(rng, max(0, n))]
        run_plan(d)
    c = plan_case(rng, 4, 9, 16, None)
    c["new"][1] = 2 ** 31 - 1
    run_plan(c)


@gpu
def test_plan_refuses_trees_of_more_tokens_than_the_mask_has_bits():
    """33 and 70 tokens where the rows have a word: what they need is not taken, and the others are as without them."""
    _, paged = mods()
    new, most = [5, 33, 32, 70, 1], 20
    lens, table = [0, 16, 3, 0, 40], [[-1] * 8 for _ in new]
    parents = [i - 1 for n in new for i in range(n)]
    free, t = list(range(30)), i32(table)
    got = paged.plan(t, i32(lens), i32(new), 16, sum(new), held=i32([0] * 5), free_pages=i32(free), free_count=i32([30]), parents=i32(parents), max_new=most)
    served = [True, False, True, False, True]
    assert got.cu_new.tolist() == [0, 5, 38, 70, 140, 141]
    assert got.seq_lens.tolist() == [c + n if ok else 0 for c, n, ok in zip(lens, new, served)]
    need = [-(-(c + n) // 16) if ok else 0 for c, n, ok in zip(lens, new, served)]
    assert got.held.tolist() == need and got.free_count.item() == 30 - sum(need)
    slots, cu = got.slots.tolist(), got.cu_new.tolist()
    at = 30
    for s, (c, n) in enumerate(zip(lens, new)):
        pages = [free[at - 1 - j] for j in range(need[s])]
        at -= need[s]
        assert t[s].tolist() == pages + [-1] * (8 - need[s])
        want = [pages[(c + i) // 16] * 16 + (c + i) % 16 for i in range(n)] if served[s] else [-1] * n
        assert slots[cu[s]:cu[s + 1]] == want
        if served[s]:
            assert torch.equal(got.mask[cu[s]:cu[s + 1]], words_of(ancestors(parents[cu[s]:cu[s + 1]]), 1))


@gpu
def test_plan_over_its_own_inputs_captured_and_on_another_stream():
    """held, free_count and the lengths in place, step after step, as a captured loop has them."""
    _, paged = mods()
    rng = random.Random(5)
    c = plan_case(rng, 70, 40, 16, "tree", spare_pages=900)
    c["table"] = [r + [-5] * 40 for r in c["table"]]
    table, lens, new, held = (i32(c[k]) for k in ("table", "lens", "new", "held"))
    free, count, parents = i32(c["free"]), i32([len(c["free"])]), i32(c["parents"])
    blank = paged.plan(table.clone(), lens, new, 16, c["tokens"], held=held, free_pages=free, free_count=count, parents=parents, max_new=c["most"])
    out = blank._replace(held=held, free_count=count, seq_lens=lens)

    def step():
        return paged.plan(table, lens, new, 16, c["tokens"], held=held, free_pages=free, free_count=count, parents=parents,
                          max_new=c["most"], out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    want, rows = plain_plan(c["table"], c["lens"], c["new"], 16, c["tokens"], c["held"], c["free"], len(c["free"]), c["parents"], blank.mask.shape[1])
    check_plan(out, want, table, rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        before = (table.tolist(), lens.tolist(), held.tolist(), count.item())
        graph.replay()
        torch.cuda.synchronize()
        want, rows = plain_plan(before[0], before[1], c["new"], 16, c["tokens"], before[2], c["free"], before[3], c["parents"], blank.mask.shape[1])
        check_plan(out, want, table, rows)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(28, 4, 128), (14, 2, 64), (4, 4, 128)])
def test_trees_past_max_new_that_the_mask_holds(dtype, nh, nkv, hd):
    """A plan for 20 tokens serves trees of 21 to 32; with the mask's bits as their bound attention and acceptance take them whole."""
    _, paged = mods()
    rng = random.Random(6)
    new, ctx = [32, 5, 33, 21], [400, 5, 90, 1000]
    q, cache, table, lens, cu = build(gen(4), new, ctx, nh, nkv, hd, 16, dtype)
    parents = [p for n in new for p in tree(rng, n)]
    p = paged.plan(table, lens - i32(new), i32(new), 16, sum(new), parents=i32(parents), max_new=20)
    assert p.seq_lens.tolist() == [400, 5, 0, 1000] and p.mask.shape[1] == 1
    y = paged.tree_attention(q, cache, table, p.seq_lens, p.cu_new, p.mask, max_new=32 * p.mask.shape[1])
    at = p.cu_new.tolist()
    y[at[2] + 32] = 0   # the refused tree's last row, past the bound, is left unwritten
    sees = [see_of(ancestors(parents[a:b]) if c else [0] * (b - a), c, b - a) for a, b, c in zip(at, at[1:], p.seq_lens.tolist())]
    check_tree(q, cache, table, p.seq_lens.tolist(), new, sees, y, 1 / math.sqrt(hd))
    x = randn(gen(5), sum(new), 300, dtype=dtype)
    tokens = i64([x[a + max(0, parents[a + i])].argmax().item() for a, b in zip(at, at[1:]) for i in range(b - a)])
    got = paged.verify(x, tokens, i32(parents), p.cu_new, max_new=32, seq_lens=p.seq_lens)
    want = plain_verify(x, tokens.tolist(), parents, new, 32)
    for s in range(4):
        if s == 2:
            assert got.accepted[s] == 0 and got.next[s] == -1
        else:
            assert got.accepted[s] == want[0][s] and torch.equal(got.path[s], want[1][s]) and got.next[s] == want[2][s]
    looked_at = [i for i in range(sum(new)) if i != at[2] + 32]   # (the refused tree's last row is past the bound)
    assert torch.equal(got.targets[looked_at], want[3][looked_at]) and status() == 0


@gpu
def test_plans_of_different_sizes_at_once():
    """From two host threads, of so many sequences that the kernel's shared memory is more than what it has by default: neither call
    takes from the other what it may use."""
    _, paged = mods()
    faults, together = [], threading.Barrier(3)

    def work(seqs):
        try:
            table, lens, new = torch.zeros(seqs, 1, dtype=torch.int32, device="cuda"), i32([3] * seqs), i32([1] * seqs)
            out = paged.plan(table, lens, new, 16, seqs)
            with torch.cuda.stream(torch.cuda.Stream()):
                together.wait(60)
                for _ in range(10000):
                    paged.plan(table, lens, new, 16, seqs, out=out)
                torch.cuda.current_stream().synchronize()
            assert out.cu_new.tolist() == list(range(seqs + 1)) and out.slots.tolist() == [3] * seqs
        except Exception as e:   # (an assertion in a thread would be lost)
            faults.append(e)

    threads = [threading.Thread(target=work, args=(seqs,)) for seqs in (8192, 4000, 6000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not faults, faults


@gpu
def test_a_captured_plan_of_many_sequences_after_a_smaller_one():
    _, paged = mods()
    made = []
    for seqs in (8192, 3500):
        args = torch.zeros(seqs, 1, dtype=torch.int32, device="cuda"), i32([3] * seqs), i32([1] * seqs), 16, seqs
        out, graph = paged.plan(*args), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged.plan(*args, out=out)
        made.append((seqs, out, graph, args))   # (a graph keeps no inputs alive)
    for _ in range(3):
        for seqs, out, graph, _ in made:
            out.slots.fill_(-9), out.cu_new.fill_(-9)
            graph.replay()
            assert out.cu_new.tolist() == list(range(seqs + 1)) and out.slots.tolist() == [3] * seqs


@gpu
@pytest.mark.parametrize("inference", [False, True])
def test_outputs_of_plan_and_verify_do_not_share_values(inference):
    """Filled one after another, each keeps its own; sizes that end off every boundary; inside inference mode too."""
    _, paged = mods()
    rng = random.Random(8)
    c = plan_case(rng, 7, 40, 16, "tree", spare_tokens=3)
    with torch.inference_mode(inference):
        got = run_plan(c)
        x = randn(gen(1), 13, 1001, dtype=torch.float16)
        ok = paged.verify(x, i64([0] * 13), i32([-1] + list(range(12))), i32([0, 5, 13]), max_path=3)
        for outs in (got, ok):
            for i, t in enumerate(outs):
                assert t.is_contiguous() and not t.requires_grad and t.is_inference() == inference
                t.fill_(100 + i)
            torch.cuda.synchronize()
            assert all((t == 100 + i).all() for i, t in enumerate(outs))
            assert [t.clone().numel() for t in outs] == [t.numel() for t in outs]


@gpu
def test_plan_refusals():
    _, paged = mods()
    table, v = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), i32([1, 2, 3])
    ok = dict(page_table=table, seq_lens=v, new_lens=v, page_size=16, tokens=6)
    paged.plan(**ok)
    paged.plan(**dict(ok, tokens=0, new_lens=i32([0, 0, 0])))
    for kw in (dict(page_table=table.long()), dict(page_table=table.cpu()), dict(page_table=table[:0]), dict(page_table=table.t()), dict(seq_lens=v[:2]),
               dict(seq_lens=v.long()), dict(new_lens=v.cpu()), dict(page_size=24), dict(page_size=0), dict(tokens=-1), dict(held=v),
               dict(held=v, free_pages=v), dict(free_count=i32([1])), dict(held=v, free_pages=v, free_count=v),
               dict(parents=v), dict(parents=i64([0] * 6)), dict(out=paged.plan(**ok)._replace(slots=v))):
        with pytest.raises(RuntimeError):
            paged.plan(**{**ok, **kw})
    with pytest.raises(ValueError, match="1024"):
        paged.plan(**ok, parents=i32([0] * 6), max_new=1025)


# ------------------------------------------------------------------------------------------------- tree attention

def see_of(rows, ctx, new):
    """[n, ctx] truth values of one sequence: what its new tokens see."""
    see = torch.ones(new, ctx, dtype=torch.bool)
    first = max(0, ctx - new)   # the first key that is a new token's
    if ctx and new:
        see[:, first:] = torch.tensor([[bool(r >> key - (ctx - new) & 1) for key in range(first, ctx)] for r in rows], dtype=torch.bool).view(new, -1)
    return see.cuda()


def check_tree(q, cache, table, ctx, new, sees, y, scale):
    nh, hd = q.shape[1:]
    grp, u, t = nh // cache.nkv, U[q.dtype], 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        if not n:
            continue
        if c:
            pages = table[s, : -(-c // cache.page_size)].long()
            k, v = (x[pages].permute(0, 2, 1, 3).reshape(-1, cache.nkv, hd)[:c].double().repeat_interleave(grp, 1)
                    for x in (cache.k, cache.v))
            score = torch.einsum("nhd,khd->hnk", q[t:t + n].double(), k) * scale
            p = torch.nan_to_num(torch.softmax(score.masked_fill(~sees[s], float("-inf")), -1), nan=0.0)
            want, absv = torch.einsum("hnk,khd->nhd", p, v), torch.einsum("hnk,khd->nhd", p, v.abs())
            tol = u * want.abs() + (1.25 * u + 2.0 ** -12) * absv + (c * 2.0 ** -25 * v.abs().amax() if q.dtype == torch.float16 else 0)
            close(y[t:t + n], want, tol, f"new={n} ctx={c}")
            blind = ~sees[s].any(1)
            assert (y[t:t + n][blind] == 0).all()
        else:
            assert (y[t:t + n] == 0).all()
        t += n


def bits_for(rng, kind, n):
    if kind == "tree":
        return ancestors(tree(rng, n))
    if kind == "chain":
        return [(1 << i + 1) - 1 for i in range(n)]
    if kind == "none":
        return [0] * n
    return [rng.getrandbits(n) if rng.random() < 0.8 else 0 for _ in range(n)]   # any pattern, bits past themselves too


def run_tree(seed, new, ctx, nh, nkv, hd, page, dtype, kind, words=None, **kw):
    _, paged = mods()
    q, cache, table, lens, cu = build(gen(seed), new, ctx, nh, nkv, hd, page, dtype)
    rng = random.Random(seed)
    rows = [bits_for(rng, kind, n) for n in new]
    words = -(-max(new + [1]) // 32) if words is None else words
    junk = [rng.getrandbits(1024) << n for n in new]   # bits past a sequence's new tokens stand for nothing
    mask = words_of([r | j for row, j in zip(rows, junk) for r in row], words)
    sees = [see_of([r & (1 << 32 * words) - 1 for r in row], c, n) for row, c, n in zip(rows, ctx, new)]
    y = paged.tree_attention(q, cache, table, lens, cu, mask, **kw)
    check_tree(q, cache, table, ctx, new, sees, y, kw.get("scale") or 1 / math.sqrt(hd))
    assert torch.equal(y, paged.tree_attention(q, cache, table, lens, cu, mask, **kw))   # the same bits every time
    assert status() == 0
    return q, cache, table, lens, cu, mask, y


HEADS = [(16, 2, 128), (28, 4, 128), (14, 2, 64), (4, 4, 64), (40, 1, 128), (1, 1, 128)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_tree_attention(dtype, nh, nkv, hd):
    for i, (page, new, ctx) in enumerate(((16, [1], [1]), (16, [5], [5]), (32, [8, 3], [70, 3]), (64, [17], [64]), (48, [40], [300]),
                                          (256, [64, 1, 0, 130], [64, 77, 20, 700]), (128, [33], [129]), (16, [255], [1111]),
                                          (80, [31, 2, 33], [600, 1500, 33]), (16, [8, 8, 8, 5], [900, 17, 8, 130]))):
        for kind in ("tree", "random"):
            run_tree(nh + hd + i, new, ctx, nh, nkv, hd, page, dtype, kind)
            run_tree(nh + hd + i, new, ctx, nh, nkv, hd, page, dtype, kind, max_new=max(new), max_len=max(ctx))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,ctx", [([5], [3]), ([40, 3], [7, 0]), ([1, 1, 1], [0, 0, 4]), ([0, 1], [9, 1]), ([200], [130]), ([6], [6]), ([129], [129])])
def test_tree_attention_rows_that_see_nothing(dtype, new, ctx):
    """Masks without a bit over no context, and lengths shorter than the new tokens (as of a refused sequence)."""
    for hd, nh, nkv in ((64, 6, 2), (128, 16, 2), (128, 40, 1)):
        for kind in ("none", "random"):
            run_tree(sum(ctx), new, ctx, nh, nkv, hd, 16, dtype, kind)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(28, 4, 128), (14, 2, 64)])
def test_tree_attention_split_contexts_and_ragged_batches(dtype, nh, nkv, hd):
    """Clusters and second kernels over one long context; more sequences than a warp; masks of few words."""
    rng = random.Random(nh)
    for new, ctx in (([4], [20000]), ([60], [9000]), ([300], [4000])):
        run_tree(7, new, ctx, nh, nkv, hd, 64, dtype, "tree", max_new=new[0])
    for n in (8, 61):
        new = [rng.choice((0, 1, n, rng.randint(1, n))) for _ in range(67)]
        new[5] = n
        run_tree(8, new, [m + rng.randint(0, 500) for m in new], nh, nkv, hd, 16, dtype, "tree", max_new=n)
    run_tree(9, [61, 90], [300, 400], nh, nkv, hd, 16, dtype, "random", words=1)   # tokens past the words are seen by none
    run_tree(9, [61, 9], [300, 400], nh, nkv, hd, 16, dtype, "random", words=32)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,ctx,nh,nkv,hd", [([64], [5000], 16, 2, 128), ([200], [9001], 14, 2, 64), ([61, 10, 0, 5], [6000, 12, 70, 0], 16, 2, 128), ([33], [1000], 8, 2, 64),
                                               ([255], [20001], 28, 4, 128), ([1000], [1000], 2, 2, 128), ([70, 3], [3, 3000], 4, 4, 64)])
def test_tree_attention_contexts_split_through_the_workspace(dtype, new, ctx, nh, nkv, hd):
    """More CTAs a context than a cluster has; parts without keys, rows that see nothing in any or in all of them."""
    ops, paged = mods()
    for kind in ("tree", "any", "none"):
        q, cache, table, lens, cu, mask, y = run_tree(21, new, ctx, nh, nkv, hd, 16, dtype, kind, max_new=max(new), max_len=max(ctx))
        t, w = q.shape[0], table.shape[1]
        assert ops.ext().lib.lb_paged_tree_attention_workspace(t, nh, cache._ptr, w, len(new), max(new), max(ctx)) > 0
        graph, out = torch.cuda.CUDAGraph(), torch.full_like(y, 5.0)
        with torch.cuda.graph(graph):
            paged.tree_attention(q, cache, table, lens, cu, mask, max_new=max(new), max_len=max(ctx), out=out)
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, y)
    assert status() == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_attention_up_to_128_rows_over_many_key_tiles(dtype):
    """Odd and even counts of key tiles, from one CTA a context to clusters and the workspace; contexts and parts without keys, rows
    that see nothing; 128 rows and one."""
    rng = random.Random(3)
    for nh, nkv, new, ctx in ((28, 4, [18] * 40, [rng.randint(18, 1100) for _ in range(40)]), (16, 2, [16, 3, 1, 0, 16, 16], [5000, 129, 0, 8, 640, 641]),
                              (28, 4, [18], [12000]), (28, 4, [9], [129]), (8, 8, [128], [3000]), (8, 8, [100, 128, 1], [1281, 2305, 1153]),
                              (32, 4, [16] * 70, [16 + 37 * i for i in range(70)]), (16, 2, [16] * 12, [16 + 700 * i for i in range(12)])):
        for kind in ("tree", "any", "none"):
            run_tree(41, new, ctx, nh, nkv, 128, 16, dtype, kind, max_new=max(new), max_len=max(ctx))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(28, 4, 128), (16, 2, 128), (14, 2, 64), (8, 8, 128)])
def test_tree_attention_small_trees_whichever_kernel_takes_them(dtype, nh, nkv, hd):
    """1 to 64 rows a key head, where contexts and batches decide between the kernels; single tokens and empty contexts among them."""
    rng = random.Random(nh + hd)
    for seqs, most, longest in ((1, 8, 9000), (1, 4, 9000), (24, 8, 3000), (24, 4, 700), (70, 3, 900), (40, 1, 2000), (5, 8, 200)):
        new = [rng.choice((most, rng.randint(0, most))) for _ in range(seqs)]
        ctx = [rng.choice((longest, rng.randint(n, longest), n)) for n in new]
        new[0], ctx[0] = most, longest
        if seqs > 2:
            new[-1], ctx[-1] = 1, 0
        for kind in ("tree", "any"):
            run_tree(31, new, ctx, nh, nkv, hd, 16, dtype, kind, max_new=most, max_len=longest)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,ctx", [(3, 40), (8, 300), (60, 300), (200, 900)])
def test_tree_attention_of_a_chain_is_attention(dtype, n, ctx):
    """A chain's mask is the causal one: the same values to the roundings of two orders of the sums."""
    _, paged = mods()
    for nh, nkv, hd in ((16, 2, 128), (14, 2, 64)):
        q, cache, table, lens, cu, mask, y = run_tree(3, [n], [ctx], nh, nkv, hd, 32, dtype, "chain", max_new=n)
        other = paged.attention(q, cache, table, lens, cu, max_new=n)
        assert ((y.double() - other.double()).abs() <= 8 * U[dtype] * (1 + other.double().abs())).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [6, 100])
def test_tree_attention_unseen_keys_have_no_weight(dtype, n):
    """K rows of NaN and infinity, V rows at the end of the type's range: tokens whose bit is not set are bit for bit as they were."""
    _, paged = mods()
    q, cache, table, lens, cu, mask, clean = run_tree(12, [n], [300], 16, 2, 128, 32, dtype, "tree", max_new=n)
    bits = [[(int(mask[i, j // 32]) >> j % 32) & 1 for j in range(n)] for i in range(n)]
    for j in (1, 2, n // 2, n - 1):
        key = 300 - n + j
        at, row = int(table[0, key // 32]), key % 32
        blind = torch.tensor([not bits[i][j] for i in range(n)], device="cuda")
        for t, v in ((cache.k, float("nan")), (cache.k, float("inf")), (cache.v, -0.9 * torch.finfo(dtype).max)):
            keep = t[at, :, row].clone()
            t[at, :, row] = v
            y = paged.tree_attention(q, cache, table, lens, cu, mask, max_new=n)
            assert torch.equal(y[blind], clean[blind]), j
            if t is cache.k and v != v:
                assert torch.isnan(y[~blind]).all()
            t[at, :, row] = keep


@gpu
def test_tree_attention_strides_padding_and_graph():
    _, paged = mods()
    new, ctx = [9, 30, 1], [100, 250, 40]
    q, cache, table, lens, cu, mask, y = run_tree(5, new, ctx, 8, 2, 128, 16, torch.float16, "tree", max_new=30)
    wide = torch.zeros(40, 10, 192, device="cuda", dtype=torch.float16)
    wide[:, 1:9, 32:160] = 7
    wide[:40, 1:9, 32:160] = q
    assert torch.equal(paged.tree_attention(wide[:, 1:9, 32:160], cache, table, lens, cu, mask, max_new=30), y)
    padded, rows = torch.cat((q, q[:5])), torch.cat((mask, mask[:5]))
    out = torch.full((45, 8, 128), 3.0, device="cuda", dtype=torch.float16)
    paged.tree_attention(padded, cache, table, lens, cu, rows, max_new=30, out=out)
    assert torch.equal(out[:40], y) and (out[40:] == 3).all()
    graph, got = torch.cuda.CUDAGraph(), torch.zeros_like(y)
    with torch.cuda.graph(graph):
        paged.tree_attention(q, cache, table, lens, cu, mask, max_new=30, out=got)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, y)
    mask.copy_(words_of([(1 << i + 1) - 1 for n in new for i in range(n)], 1))   # read at the replay
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = paged.tree_attention(q, cache, table, lens, cu, mask, max_new=30)
    side.synchronize()
    assert torch.equal(got, again) and not torch.equal(got, y)


@gpu
def test_tree_attention_refusals():
    _, paged = mods()
    q, cache, table, lens, cu = build(gen(4), [2, 1], [20, 9], 4, 2, 64, 16, torch.float16)
    mask = torch.ones(3, 1, dtype=torch.int32, device="cuda")
    ok = dict(q=q, cache=cache, page_table=table, seq_lens=lens, cu_new=cu, mask=mask)
    paged.tree_attention(**ok)
    for kw in (dict(mask=None), dict(mask=mask.long()), dict(mask=mask[:2]), dict(mask=mask[:, 0]), dict(mask=mask[:, :0]), dict(mask=mask.cpu()),
               dict(mask=torch.ones(3, 2, dtype=torch.int32, device="cuda")[:, :1]), dict(q=q.bfloat16()), dict(max_new=0), dict(scale=0.0),
               dict(seq_lens=lens[:1]), dict(cu_new=cu[:2]), dict(page_table=table[0])):
        with pytest.raises(RuntimeError):
            paged.tree_attention(**{**ok, **kw})


# --------------------------------------------------------------------------------------------------------- verify

def plain_verify(logits, tokens, parents, new, max_path):
    best = []
    for row in logits.double().cpu():
        nan = torch.isnan(row)
        best.append(int(nan.int().argmax()) if nan.any() else int((row == row.max()).int().argmax()))
    accepted, paths, after, at = [], [], [], 0
    for n in new:
        path = [0] if n else []
        while path and len(path) < max_path:
            child = [c for c in range(path[-1] + 1, n) if parents[at + c] == path[-1] and tokens[at + c] == best[at + path[-1]]]
            if not child:
                break
            path.append(child[0])
        accepted.append(len(path))
        after.append(best[at + path[-1]] if path else -1)
        paths.append(path + [-1] * (max_path - len(path)))
        at += n
    return i32(accepted), i32(paths), i64(after), i64(best[:at])


def check_verify(logits, tokens, parents, new, max_path=None, **kw):
    _, paged = mods()
    most = kw.get("max_new") or sum(new)
    got = paged.verify(logits, i64(tokens), i32(parents), cu_of(new), max_path=max_path, **kw)
    want = plain_verify(logits, tokens, parents, new, max_path or most)
    for name, g, w in zip(got._fields, got, want):
        if name == "targets":
            g = g[:len(w)]
        assert torch.equal(g, w), name
    return got


def drafts(rng, logits, new, p=0.7):
    """Trees over those logits: a child is its parent's target with that chance."""
    top, tokens, parents, at = logits.float().nan_to_num(nan=1e30).argmax(1).tolist(), [], [], 0
    for n in new:
        shape = tree(rng, n)
        tokens += [top[at + q] if q >= 0 and rng.random() < p else rng.randrange(logits.shape[1]) for q in shape]
        parents += shape
        at += n
    return tokens, parents


@gpu
@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 1000, 8191, 32003, 151936, 200001])
def test_verify(dtype, vocab):
    rng = random.Random(vocab)
    for new in ([1], [8], [1, 31, 0, 17], [3] * 40):
        logits = randn(gen(vocab), sum(new), vocab, dtype=dtype)   # 16-bit values: many largest ones are equal
        tokens, parents = drafts(rng, logits, new)
        check_verify(logits, tokens, parents, new)
        check_verify(logits, tokens, parents, new, max_new=max(new), max_path=3)
    assert status() == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
def test_verify_strides_and_special_values(dtype):
    """Rows that start anywhere; NaN, infinities, zeros of both signs and constant rows, the first of equal values each time."""
    rng = random.Random(3)
    for vocab, pad in ((1001, 3), (40000, 5), (4096, 1), (9, 2)):
        big = randn(gen(vocab), 24, vocab + pad, dtype=dtype)
        for off in range(pad):
            x = big[:, off:off + vocab]
            x[0] = float("-inf")
            x[1] = 0.0
            x[1, vocab // 2:] = -0.0
            x[2] = -0.0
            x[2, vocab // 3:] = 0.0
            x[3, vocab - 1] = float("nan")
            x[4, vocab // 2], x[4, 1] = float("nan"), float("inf")
            x[5, 1:] = float("inf")
            x[6] = torch.finfo(dtype).min
            x[7] = float("-inf")
            x[7, vocab - 1] = torch.finfo(dtype).min
            tokens, parents = drafts(rng, x, [24], 0.9)
            check_verify(x, tokens, parents, [24])


@gpu
def test_verify_trees():
    """Chains that are all accepted, up to 1024 tokens; children that are equal, that come before their parent, that are their own
    parents; parents outside the tree; bounds below the truth."""
    _, paged = mods()
    x = randn(gen(1), 1024, 300, dtype=torch.float16)
    top = x.float().argmax(1).tolist()
    chain = list(range(-1, 1023))
    got = check_verify(x, [5] + top[:-1], chain, [1024])
    assert got.accepted.item() == 1024
    check_verify(x, [5] + top[:-1], chain, [1024], max_path=1)
    check_verify(x, [5] + top[:-1], chain, [1024], max_path=700)
    check_verify(x[:6], [1, top[0], top[0], top[1], top[2], 9], [-1, 0, 0, 1, 2, 4], [6])        # the first of two equal children
    check_verify(x[:5], [1, top[0], top[1], top[3], 3], [-1, 0, 3, 1, -7], [5])                   # 2's parent comes after it
    check_verify(x[:4], [top[0], top[0], top[1], top[2]], [0, 1, 2, 99], [4])                     # its own parent
    check_verify(x[:70], [1] + [3] * 66 + [top[0], top[67], top[68]], [-1] + [0] * 67 + [67, 68], [70])
    got = paged.verify(x[:40], i64([5] + top[:39]), i32(list(range(-1, 39))), i32([0, 20, 40]), max_new=8)   # those behind the bound are ignored
    assert got.accepted.tolist() == [8, 1] and got.path.shape == (2, 8)
    empty = paged.verify(x[:0], i64([]), i32([]), i32([0, 0]))
    assert empty.accepted.tolist() == [0] and empty.next.tolist() == [-1]


@gpu
@pytest.mark.parametrize("contiguous", [True, False])
def test_verify_accepts_nothing_for_sequences_that_the_plan_refused(contiguous):
    """With the plan's lengths, whether the refused one has all, some or none of its rows; the others are as without them."""
    _, paged = mods()
    new, vocab = [6, 9, 4, 0, 7, 5], 500
    x = randn(gen(3), 31, vocab, dtype=torch.float16)
    if not contiguous:   # (rows that the checked path has to lay out first)
        x = x.t().contiguous().t()
    top = x.argmax(1).tolist()
    tokens, parents = [t for i in range(31) for t in ([7] if i in (0, 6, 15, 19, 26) else [top[i - 1]])], [i - 1 for n in new for i in range(n)]
    table, before = i32([[2 * i, 2 * i + 1] for i in range(6)]), i32([10, 30, 3, 0, 0, 2])
    for rows, served in ((31, [1, 0, 1, 1, 1, 1]), (23, [1, 0, 1, 1, 0, 0]), (19, [1, 0, 1, 1, 0, 0])):
        at = paged.plan(table, before, i32(new), 16, rows, parents=i32(parents[:rows]), max_new=9)
        assert [int(n > 0 or i == 3) for i, n in enumerate(at.seq_lens.tolist())] == served
        args = x[:rows], i64(tokens[:rows]), i32(parents[:rows]), at.cu_new
        plain, got = paged.verify(*args, max_new=9), paged.verify(*args, max_new=9, seq_lens=at.seq_lens)
        assert torch.equal(got.targets, plain.targets)
        for s, ok in enumerate(served):
            if ok:
                assert torch.equal(got.path[s], plain.path[s]) and (got.accepted[s], got.next[s]) == (plain.accepted[s], plain.next[s])
            else:
                assert got.accepted[s] == 0 and got.next[s] == -1 and (got.path[s] == -1).all()
    # fewer new tokens looked at than there are: refused by all of them
    got = paged.verify(*args, max_new=2, seq_lens=i32([5, 8, 4, 0, 0, 0]))
    assert got.accepted.tolist() == [0, 0, 2, 0, 0, 0]
    for bad in (i32([1] * 5), i64([1] * 6), torch.zeros(6, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="seq_lens"):
            paged.verify(*args, seq_lens=bad)


@gpu
def test_verify_leaves_rows_behind_the_last_sequence_and_replays():
    _, paged = mods()
    rng = random.Random(2)
    new, spare = [9, 4], 7
    x = randn(gen(8), 20, 5000, dtype=torch.bfloat16)
    x[13:] = float("nan")
    tokens, parents = drafts(rng, x[:13], new)
    t, p, cu = i64(tokens + [0] * spare), i32(parents + [0] * spare), cu_of(new)
    graph = torch.cuda.CUDAGraph()
    paged.verify(x, t, p, cu, max_new=9)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = paged.verify(x, t, p, cu, max_new=9)
    for seed in (1, 2, 3):
        x[:13] = randn(gen(seed), 13, 5000, dtype=torch.bfloat16)
        tokens, parents = drafts(rng, x[:13], new)
        t[:13], p[:13] = i64(tokens), i32(parents)
        got.targets.fill_(-9)
        graph.replay()
        want = plain_verify(x[:13], tokens, parents, new, 9)
        assert all(torch.equal(a, b) for a, b in zip(got[:3], want[:3])) and torch.equal(got.targets[:13], want[3])
        assert (got.targets[13:] == -9).all()


@gpu
def test_verify_refusals():
    _, paged = mods()
    x = torch.zeros(4, 100, device="cuda")
    ok = dict(logits=x, tokens=i64([0] * 4), parents=i32([0] * 4), cu_new=i32([0, 4]))
    paged.verify(**ok)
    paged.verify(**dict(ok, logits=x.t().contiguous().t()))
    for kw in (dict(logits=x.double()), dict(logits=x.cpu()), dict(logits=x[0]), dict(logits=x[:, :0]), dict(tokens=i32([0] * 4)), dict(tokens=i64([0] * 3)),
               dict(parents=i64([0] * 4)), dict(cu_new=i64([0, 4])), dict(cu_new=i32([0])), dict(cu_new=i32([[0, 4]]))):
        with pytest.raises(RuntimeError):
            paged.verify(**{**ok, **kw})
    for kw in (dict(max_new=0), dict(max_new=1025), dict(max_path=0), dict(max_path=1025)):
        with pytest.raises(ValueError):
            paged.verify(**{**ok, **kw})


# -------------------------------------------------------------------------------------------------------- compact

def rising(rng, n, most):
    """A path from token 0 up through some of n tokens, its sources among its destinations too."""
    path = [0]
    while len(path) < most and path[-1] + 1 < n and rng.random() < 0.9:
        path.append(rng.randint(path[-1] + 1, min(n - 1, path[-1] + 3)))
    return path


def make_caches(g, layers, pages, nkv, page, hd, dtype):
    _, paged = mods()
    both = [randn(g, pages, 2, nkv, page, hd, dtype=dtype) for _ in range(layers)]
    return [paged.PagedCache.from_tensors(b[:, 0], b[:, 1]) for b in both]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers,nkv,hd,page", [(1, 1, 64, 16), (3, 2, 128, 48), (36, 2, 128, 16), (2, 5, 16, 32), (2, 3, 48, 16), (128, 1, 256, 64)])
def test_compact(dtype, layers, nkv, hd, page):
    _, paged = mods()
    rng = random.Random(layers + hd)
    for new, most in (([1], 4), ([9, 0, 30, 1], 12), ([700], 600), ([20] * 30, 9)):
        if layers * len(new) > 200 or layers * max(new) > 30000:
            continue
        ctx = [n + rng.choice((0, 3, page, 5 * page - 1)) for n in new]
        need = [-(-c // page) for c in ctx]
        pages = sum(need) + 2
        caches = make_caches(gen(hd), layers, pages, nkv, page, hd, dtype)
        order = list(range(pages))
        rng.shuffle(order)
        table = [[order.pop() for _ in range(k)] for k in need]
        width = max(need + [1]) + 1
        paths = [rising(rng, n, most) if n else [] for n in new]
        want = [(c.k.clone(), c.v.clone()) for c in caches]
        for s, path in enumerate(paths):
            start = ctx[s] - new[s]
            for d, i in enumerate(path):
                a, b = start + i, start + d
                for pair in want:
                    for t in pair:
                        t[table[s][b // page], :, b % page] = t[table[s][a // page], :, a % page]
        lens = paged.compact(caches, i32([r + [-1] * (width - len(r)) for r in table]), i32(ctx), cu_of(new),
                             i32([p + [-1] * (most - len(p)) for p in paths]), i32([len(p) for p in paths]))
        assert lens.tolist() == [c - n + len(p) for c, n, p in zip(ctx, new, paths)]
        for c, (k, v) in zip(caches, want):
            assert torch.equal(c.k, k) and torch.equal(c.v, v)
    assert status() == 0


@gpu
def test_compact_leaves_refused_sequences_and_reports_bad_paths():
    ops, paged = mods()
    lib = ops.ext().lib
    caches = make_caches(gen(1), 2, 8, 2, 16, 64, torch.float16)
    table = i32([[0, 1], [2, 3], [4, 9]])
    keep = [(c.k.clone(), c.v.clone()) for c in caches]
    lens, cu, path, count = i32([0, 20, 30]), cu_of([4, 5, 20]), i32([[0, 2, 3], [0, 1, 2], [0, 1, 2]]), i32([3, 3, 3])
    out = i32([77, 77, 77])
    assert paged.compact(caches, table, lens, cu, path, count).tolist() == [0, 18, 13]
    assert paged.compact(caches, table, lens, cu, path, count, out=out) is out and out.tolist() == [77, 18, 13]
    assert all(torch.equal(c.k, k) and torch.equal(c.v, v) for c, (k, v) in zip(caches, keep))   # paths that stay in place
    assert lib.lb_device_error() == 0
    try:
        for bad in ([[0, 0, 0], [0, 1, 0], [0, 1, 2]], [[0, 0, 0], [0, 5, 2], [0, 1, 2]], [[0, 0, 0], [0, 2 ** 31 - 1, 2], [0, 1, 2]],
                    [[0, 0, 0], [0, 1, 2], [0, 7, 2]]):   # below its place, past the new tokens, on a page outside the cache
            paged.compact(caches, table, lens, cu, i32(bad), count)
            assert lib.lb_device_error() == 3
            lib.lb_clear_device_error()
        assert all(torch.equal(c.k, k) and torch.equal(c.v, v) for c, (k, v) in zip(caches, keep))
    finally:
        lib.lb_clear_device_error()


@gpu
@pytest.mark.parametrize("short", ["rows", "width", "pages"])
def test_compact_keeps_the_lengths_of_all_sequences_that_the_plan_refused(short):
    """Those behind the one that did not fit have no rows left, so that nothing but their length, 0, says that they were refused; served
    ones without new tokens and empty ones are as they were."""
    _, paged = mods()
    caches = make_caches(gen(1), 2, 160, 2, 16, 64, torch.float16)
    table = torch.randperm(160, device="cuda", generator=gen(2))[:140].view(7, 20).to(torch.int32)
    before, new, kw = [100, 200, 300, 0, 5, 60, 90], [8, 8, 8, 0, 0, 3, 0], {}
    tokens = sum(new)
    if short == "rows":   # four for the second sequence, none for the third and the sixth
        tokens, served = 12, [True, False, False, True, True, False, True]
    elif short == "width":   # contexts up to 112; the second one asks for nothing
        new[1], served = 0, [True, False, False, True, True, True, True]
        table, tokens = table[:, :7].contiguous(), sum(new)
    else:   # no page is free, the third and the last sequence need one
        before[2], before[6], new[6] = 304, 95, 2
        kw = dict(held=i32([7, 13, 19, 0, 1, 4, 6]), free_pages=i32([159]), free_count=i32([0]))
        tokens, served = sum(new), [True, True, False, True, True, True, False]
    lens = i32(before)
    p = paged.plan(table, lens, i32(new), 16, tokens, **kw)
    assert p.seq_lens.tolist() == [c + n if ok else 0 for c, n, ok in zip(before, new, served)]
    if short == "rows":
        assert p.cu_new.tolist() == [0, 8, 12, 12, 12, 12, 12, 12]
    path, count = i32([[0, 1, 2] if n else [-1] * 3 for n in new]), i32([min(n, 3) for n in new])
    kept = [(c.k.clone(), c.v.clone()) for c in caches]
    want = [c + min(n, 3) if ok else 0 for c, n, ok in zip(before, new, served)]
    assert paged.compact(caches, table, p.seq_lens, p.cu_new, path, count).tolist() == want
    want = [w if ok else c for w, c, ok in zip(want, before, served)]
    assert paged.compact(caches, table, p.seq_lens, p.cu_new, path, count, out=lens) is lens and lens.tolist() == want
    assert all(torch.equal(c.k, k) and torch.equal(c.v, v) for c, (k, v) in zip(caches, kept)) and status() == 0


@gpu
def test_compact_moves_a_path_that_does_not_rise_as_it_stands():
    """Every entry's row as it was before the call: each lies at or behind its own place, so no row is written before it is read."""
    _, paged = mods()
    for path in ([0, 5, 3], [0, 4, 4, 4], [0, 9, 8, 7, 6, 5], [2, 2, 2, 9, 4]):
        cache = make_caches(gen(len(path)), 1, 4, 2, 16, 64, torch.bfloat16)[0]
        rows = [t.transpose(1, 2).reshape(64, 2, 64).clone() for t in (cache.k, cache.v)]
        start = 10   # the rows 10 to 19 of pages 2 and 0
        at = lambda j: (2, 0)[(start + j) // 16] * 16 + (start + j) % 16
        want = [r.clone() for r in rows]
        for w, r in zip(want, rows):
            w[i64([at(d) for d in range(len(path))])] = r[i64([at(j) for j in path])]
        paged.compact([cache], i32([[2, 0]]), i32([20]), i32([0, 10]), i32([path]), i32([len(path)]))
        assert all(torch.equal(t.transpose(1, 2).reshape(64, 2, 64), w) for t, w in zip((cache.k, cache.v), want)) and status() == 0


@gpu
def test_compact_refusals():
    _, paged = mods()
    caches = make_caches(gen(1), 2, 8, 2, 16, 64, torch.float16)
    ok = dict(caches=caches, page_table=i32([[0, 1]]), seq_lens=i32([20]), cu_new=i32([0, 5]), path=i32([[0, 2]]), accepted=i32([2]))
    paged.compact(**ok)
    for kw in (dict(caches=[]), dict(caches=[caches[0].k]), dict(caches=caches + [paged.PagedCache(8, 16, 2, 64)]),
               dict(caches=caches + [paged.PagedCache(8, 16, 2, 64, torch.bfloat16)]), dict(caches=caches * 65), dict(page_table=i64([[0, 1]])),
               dict(seq_lens=i32([20, 1])), dict(cu_new=i32([0])), dict(path=i32([0, 2])), dict(path=i32([[]])), dict(accepted=i64([2])), dict(out=i64([2]))):
        with pytest.raises(RuntimeError):
            paged.compact(**{**ok, **kw})
    with pytest.raises(RuntimeError, match="itself"):
        paged.compact(**ok, out=ok["seq_lens"])
    buf = i32([20, 0, 5, 2])   # the output over each other input
    for kw in (dict(cu_new=buf[1:3], out=buf[2:3]), dict(accepted=buf[3:], out=buf[3:]), dict(path=buf[None, 1:3], out=buf[2:3])):
        with pytest.raises(RuntimeError, match="over an input"):
            paged.compact(**{**ok, **kw})
    with pytest.raises(RuntimeError, match="twice"):
        paged.compact(**{**ok, "caches": [caches[0], caches[1], caches[0]]})
    paged.compact(**{**ok, "accepted": buf[3:]}, out=buf[:1])
    assert buf.tolist() == [17, 0, 5, 2]


# ------------------------------------------------------------------------------------------------------ linear_f8

def f8_rule(x, dims):
    """(quantized values as fp32, scales) of x [rows, blocks, 128] or [.., 128, .., 128], a scale over `dims`."""
    amax = x.abs().amax(dims, keepdim=True).clamp(min=2.0 ** -100)
    c = torch.full_like(amax, 448.0)
    return (x * (c / amax)).to(F8).float(), amax / c


def blocks_of(w):
    n, k = w.shape
    p = torch.nn.functional.pad(w.float(), (0, -k % 128, 0, -n % 128))
    return p.view(-(-n // 128), 128, -(-k // 128), 128)


def plain_f8(x, q, scales, bias):
    """(y, A) in 64 bits: the sum, and that of the magnitudes."""
    m, k = x.shape
    n = q.shape[0]
    qx, sx = f8_rule(torch.nn.functional.pad(x.float(), (0, -k % 128)).view(m, -1, 128), 2)
    w = torch.nn.functional.pad(q.float(), (0, -k % 128)).view(n, -1, 128).double()
    t = scales.double().repeat_interleave(128, 0)[:n]
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(y)
    for b in range(w.shape[1]):
        f = sx[:, b].double() * t[:, b]
        y += qx[:, b].double() @ w[:, b].t() * f
        mag += qx[:, b].double().abs() @ w[:, b].abs().t() * f
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, mag


def check_f8(x, f8, bias, y, what=""):
    want, mag = plain_f8(x, f8.q, f8.scales, bias)
    slack = 2.0 ** -15.9 + (f8.scales.shape[1] + 3) * 2.0 ** -24
    close(y, want, U[y.dtype] * want.abs() + slack * mag, f"{what} M={x.shape[0]} K={x.shape[1]} N={f8.n}")


ROWS = [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 61, 64, 65, 100, 128, 129, 255, 256, 257, 300, 513]
WIDTHS = [(16, 1), (1, 5), (100, 37), (128, 128), (129, 130), (384, 1001), (896, 128), (2048, 256), (1000, 2000), (4864, 896)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", WIDTHS)
def test_linear_f8(dtype, k, n):
    ops, _ = mods()
    g = gen(k * 7 + n)
    f8 = ops.F8Weight.from_float(randn(g, n, k, std=0.05))
    bias = randn(g, n, dtype=dtype)
    for m in ROWS:
        x = randn(g, m, k, dtype=dtype, std=2.0)
        x[m // 2] *= 0 if m > 3 else 1
        check_f8(x, f8, None, ops.linear_f8(x, f8))
        check_f8(x, f8, bias, ops.linear_f8(x, f8, bias=bias))
    assert status() == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 300, 512), (3, 130, 384), (8, 4000, 1000), (17, 1000, 2048), (61, 4608, 3584), (70, 129, 5000), (300, 2000, 640),
                                   (629, 7531, 384), (2200, 9001, 500)])
def test_linear_f8_is_exact_where_nothing_is_rounded(dtype, m, n, k):
    """Integers that e4m3 holds, a 448 in each block so that the activations' scales are 1, weight scales that are powers of two: the sums
    are whole numbers below 2^24, and y is theirs rounded once."""
    ops, _ = mods()
    g = gen(m + n)
    x = torch.randint(-8, 9, (m, k), device="cuda", generator=g).float()
    x[:, ::128] = 448.0
    q = torch.randint(-8, 9, (n, k), device="cuda", generator=g).float()
    q[:, ::128] = torch.randint(-1, 2, q[:, ::128].shape, device="cuda", generator=g).float()
    nb, kb = -(-n // 128), -(-k // 128)
    scales = 2.0 ** torch.randint(-2, 2, (nb, kb), device="cuda", generator=g).float()
    y = ops.linear_f8((x / 64).to(dtype), ops.F8Weight(q.to(F8), scales))   # the quotient 1/64 turns up in the scales, exactly
    t = scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    want = (x.double() @ (q.double() * t).t()) / 64
    assert want.abs().max() * 256 < 2 ** 24
    assert torch.equal(y, want.to(dtype))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 16), (128, 128), (129, 257), (300, 1000), (17, 18944), (1000, 130)])
def test_quantize_f8_is_the_formula_bit_for_bit(dtype, n, k):
    ops, _ = mods()
    w = randn(gen(n + k), n, k, dtype=dtype)
    w[0, 0] = 0
    if n > 128:
        w[128:256] = 0
    if k > 128:
        w[:, 128:256] *= 1e-4
    q, s = ops.quantize_f8_gpu(w)
    want, scales = f8_rule(blocks_of(w), (1, 3))
    assert q.dtype == F8 and q.shape == (n, k) and torch.equal(s, scales[:, 0, :, 0])
    assert torch.equal(q.float(), want.reshape(want.shape[0] * 128, -1)[:n, :k])
    assert not q._base.view(torch.uint8)[:, k:].any() if q._base is not None else True


@gpu
def test_quantize_f8_of_the_smallest_and_largest_values():
    ops, _ = mods()
    for dtype, least, most in ((torch.float16, 2.0 ** -24, 65504.0), (torch.bfloat16, 2.0 ** -133, 3.3895e38), (torch.float32, 2.0 ** -149, 3.4028e38)):
        w = torch.zeros(1, 256, device="cuda", dtype=dtype)
        w[0, :3], w[0, 128:131] = torch.tensor([least, -2 * least, 4 * least]), torch.tensor([most, -most / 4, most / 8])
        q, s = ops.quantize_f8_gpu(w)
        assert q[0, 128:131].float().tolist() == [448, -112, 56]
        small = [112, -224, 448] if least > 2.0 ** -100 else [0, 0, 0]   # blocks below 2^-100 have the scale of 2^-100
        assert q[0, :3].float().tolist() == small
        assert torch.isfinite(s).all() and (s > 0).all()


@gpu
def test_linear_f8_rows_that_are_not_finite_stay_alone():
    ops, _ = mods()
    g = gen(5)
    f8 = ops.F8Weight.from_float(randn(g, 96, 384))
    for m in (4, 40, 200):
        for bad in (float("inf"), float("-inf"), float("nan")):
            x = randn(g, m, 384, dtype=torch.float16)
            clean = ops.linear_f8(x, f8)
            x[1, 200] = bad
            y = ops.linear_f8(x, f8)
            assert torch.isnan(y[1]).all()
            keep = torch.arange(m, device="cuda") != 1
            assert torch.equal(y[keep], clean[keep])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(2137, 6249, 1000), (1552, 11256, 3000), (4100, 384, 640), (700, 2000, 18944), (33, 3584, 18944), (9, 18944, 3584),
                                   (513, 128, 131072), (5, 64, 131072), (20, 40000, 130)])
def test_linear_f8_several_tiles_a_cta_and_long_rows(dtype, m, n, k):
    ops, _ = mods()
    g = gen(m)
    f8 = ops.F8Weight.from_float(randn(g, n, k, dtype=torch.bfloat16, std=0.02))
    x = randn(g, m, k, dtype=dtype)
    y = ops.linear_f8(x, f8)
    rows = torch.randint(0, m, (min(m, 150),), device="cuda", generator=g)
    check_f8(x[rows], f8, None, y[rows], f"of {m}")
    assert torch.equal(y, ops.linear_f8(x, f8)) and status() == 0


@gpu
@pytest.mark.parametrize("m,n,k", [(512, 896, 131072), (300, 224, 40000), (2048, 1792, 4096)])
def test_linear_f8_uses_each_stage_with_its_own_scale(m, n, k):
    """Tokens whose scales differ by powers of two from block to block, so that another stage's scale is off by a factor of two at least;
    small whole numbers, so that nothing is rounded before the result. Again and again, beside copies that keep memory busy."""
    ops, _ = mods()
    g = gen(k)
    blocks = -(-k // 128)
    x = torch.randint(-3, 4, (m, blocks, 128), device="cuda", generator=g).float()
    x[:, :, 0] = 7   # (a block's largest value, 448 at its scale, as are the whole numbers below it times 64)
    x = (x * 2.0 ** ((torch.arange(blocks, device="cuda") * 5 + torch.arange(m, device="cuda")[:, None]) % 8)[..., None]).view(m, -1)[:, :k].contiguous()
    w = torch.zeros(n, blocks * 128, device="cuda")
    at = torch.randint(0, blocks, (n, 40), device="cuda", generator=g) * 128 + torch.randint(0, 128, (n, 40), device="cuda", generator=g)
    w.scatter_(1, at.clamp(max=k - 1), torch.randint(-4, 5, (n, 40), device="cuda", generator=g).float())
    w = w[:, :k].contiguous()
    f8 = ops.F8Weight(w.to(F8), torch.ones(-(-n // 128), blocks, device="cuda"))
    want = x.double() @ w.double().t()   # below 2^24 in steps of 1
    x = x.to(torch.bfloat16)
    noise, side = torch.empty(1 << 26, device="cuda"), torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(side):
            noise.mul_(0.5)
        close(ops.linear_f8(x, f8), want, U[torch.bfloat16] * want.abs(), "a scale of another stage")
    assert status() == 0


@gpu
def test_linear_f8_strided_inputs_out_streams_and_graph():
    ops, _ = mods()
    g = gen(9)
    for m in (1, 6, 50, 300):
        f8 = ops.F8Weight.from_float(randn(g, 300, 500))
        wide = randn(g, m, 1300, dtype=torch.float16)
        for off in (0, 1, 3, 8):
            x = wide[:, off:off + 500]
            y = ops.linear_f8(x, f8)
            assert torch.equal(y, ops.linear_f8(x.contiguous(), f8))
            check_f8(x, f8, None, y)
        out = torch.zeros(m, 300, device="cuda", dtype=torch.float16)
        assert ops.linear_f8(x, f8, out=out) is out and torch.equal(out, y)
        assert torch.equal(ops.linear_f8(wide.t()[:500].t(), f8), ops.linear_f8(wide[:, :500], f8))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            z = ops.linear_f8(x, f8)
        side.synchronize()
        assert torch.equal(z, y)
        graph, got = torch.cuda.CUDAGraph(), torch.zeros_like(y)
        with torch.cuda.graph(graph):
            ops.linear_f8(x, f8, out=got)
        wide.copy_(randn(g, m, 1300, dtype=torch.float16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, ops.linear_f8(x, f8))
    assert ops.linear_f8(wide[:0, :500], f8).shape == (0, 300)


@gpu
@pytest.mark.parametrize("m", [1, 8, 40, 300])
def test_linear_f8_reads_weights_that_the_kernel_before_it_wrote(m):
    """Quantized in the same stream just before: neither values nor scales of the weights before may be used."""
    ops, _ = mods()
    g = gen(m)
    n, k = 2048, 2048
    x = randn(g, m, k, dtype=torch.bfloat16)
    raw = [randn(g, n, k, dtype=torch.bfloat16, std=10.0 ** -i) for i in range(3)]
    want = [ops.linear_f8(x, ops.F8Weight.from_float(w)) for w in raw]
    torch.cuda.synchronize()
    f8 = ops.F8Weight.from_float(raw[0])
    for _ in range(10):
        for w, y in zip(raw, want):
            q, s = f8.q, f8.scales
            e = ops.ext()
            assert e.lib.lb_f8_quantize_weight(w.data_ptr(), 1, n, k, k, q.data_ptr(), k, s.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
            assert torch.equal(ops.linear_f8(x, f8), y)


@gpu
@pytest.mark.parametrize("k", [64, 100])
def test_a_copy_of_an_f8_weight_is_its_own(k):
    ops, _ = mods()
    g = gen(k)
    x = randn(g, 5, k, dtype=torch.float16)
    f8 = ops.F8Weight.from_float(randn(g, 70, k))
    want = ops.linear_f8(x, f8)
    for other in (copy.deepcopy(f8), pickle.loads(pickle.dumps(f8))):
        assert torch.equal(ops.linear_f8(x, other), want)
        f8.q.view(torch.uint8).zero_()
        assert torch.equal(ops.linear_f8(x, other), want)
        f8.q.view(torch.uint8).copy_(other.q.view(torch.uint8))


@gpu
def test_linear_f8_refusals():
    ops, _ = mods()
    w = torch.ones(40, 64, device="cuda")
    f8 = ops.F8Weight.from_float(w)
    x = torch.ones(3, 64, device="cuda", dtype=torch.float16)
    for kw in (dict(x=x.float()), dict(x=x[:, :32]), dict(x=x.cpu()), dict(x=x[0]), dict(bias=torch.ones(40, device="cuda")),
               dict(bias=torch.ones(39, device="cuda", dtype=torch.float16)), dict(out=torch.ones(3, 39, device="cuda", dtype=torch.float16)),
               dict(out=torch.ones(3, 40, device="cuda", dtype=torch.bfloat16))):
        with pytest.raises(RuntimeError):
            ops.linear_f8(**{**dict(x=x, f8=f8), **kw})
    square = ops.F8Weight.from_float(torch.ones(64, 64, device="cuda"))
    with pytest.raises(RuntimeError, match="overlap"):   # other rows are still to be read when the first are written
        ops.linear_f8(x, square, out=x)
    both = torch.ones(7, 64, device="cuda", dtype=torch.float16)
    ops.linear_f8(both[:3], square, out=both[3:6])
    q, s = ops.quantize_f8_gpu(w)
    for a, b in ((q.view(torch.uint8), s), (q, s.double()), (q, s[0]), (q[0], s), (q.cpu(), s), (q, s.cpu()), (q[:0], s)):
        with pytest.raises(RuntimeError):
            ops.F8Weight(a, b)
    for bad in (w.cpu(), w.double(), w[0], w.int()):
        with pytest.raises(RuntimeError):
            ops.quantize_f8_gpu(bad)


# ------------------------------------------------------------------------------------------------------- together

@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_the_operators_give_the_same_bits_under_every_launch_option(dtype):
    ops, paged = mods()
    e = ops.ext()
    g = gen(31)
    f8 = [ops.F8Weight.from_float(randn(g, n, k, std=0.05)) for n, k in ((512, 1024), (300, 900))]
    xs = [[randn(g, m, f.k, dtype=dtype) for m in (1, 7, 40, 333)] for f in f8]
    tree_args = run_tree(2, [9, 30], [200, 300], 8, 2, 64, 16, dtype, "tree", max_new=30)
    logits = randn(g, 39, 9000, dtype=dtype)
    tokens, parents = drafts(random.Random(1), logits, [9, 30])

    def all_of_them():
        y = [ops.linear_f8(x, f) for f, row in zip(f8, xs) for x in row]
        y.append(paged.tree_attention(*tree_args[:6], max_new=30))
        return y + list(paged.verify(logits, i64(tokens), i32(parents), tree_args[4], max_new=30))

    want = all_of_them()
    try:
        for pdl in (0, 1):
            for early in (0, 1):
                e.set_option("pdl", pdl)
                e.set_option("early_weights", early)
                assert all(torch.equal(a, b) for a, b in zip(all_of_them(), want)), (pdl, early)
    finally:
        e.set_option("pdl", 1)
        e.set_option("early_weights", 0)


@gpu
@pytest.mark.parametrize("kind", ["f8", "w8"])
@pytest.mark.parametrize("m", [1, 4, 8, 40, 333])
def test_a_bias_may_come_from_the_kernel_before_under_every_launch_option(kind, m):
    """early_weights speaks of weights alone: a bias that the product before has just written is the one that is added."""
    ops, _ = mods()
    e, g = ops.ext(), gen(m)
    make, linear = (ops.F8Weight.from_float, ops.linear_f8) if kind == "f8" else (ops.W8Weight.from_float, ops.linear_w8)
    first, second = make(randn(g, 2000, 9000, std=0.05)), make(randn(g, 2000, 1024, std=0.05))
    xs, x = [randn(g, 1, 9000, dtype=torch.float16) for _ in range(8)], randn(g, m, 1024, dtype=torch.float16)
    bias = torch.empty(1, 2000, device="cuda", dtype=torch.float16)
    want = []
    for z in xs:
        linear(z, first, out=bias)
        torch.cuda.synchronize()
        want.append(linear(x, second, bias=bias[0]))
        torch.cuda.synchronize()
    try:
        for pdl in (0, 1):
            for early in (0, 1):
                e.set_option("pdl", pdl)
                e.set_option("early_weights", early)
                got = []
                for z in xs:
                    linear(z, first, out=bias)
                    got.append(linear(x, second, bias=bias[0]))
                assert all(torch.equal(a, b) for a, b in zip(got, want)), (pdl, early)
    finally:
        e.set_option("pdl", 1)
        e.set_option("early_weights", 0)


@gpu
def test_offsets_past_32_bits():
    """Pages, rows of logits and rows of tokens more than 2^31 elements from the first."""
    ops, paged = mods()
    # the attention and the move: pages 2^27 elements apart, the same bits as in a small cache
    near, stride = make_caches(gen(2), 1, 20, 2, 16, 64, torch.bfloat16)[0], 1 << 27
    room = torch.empty(19 * stride + 4096, dtype=torch.bfloat16, device="cuda")
    k, v = (room[at:].as_strided((20, 2, 16, 64), (stride, 1024, 64, 1)) for at in (0, 2048))
    k.copy_(near.k), v.copy_(near.v)
    far = paged.PagedCache.from_tensors(k, v)
    table, q = i32([list(range(19, -1, -1))]), randn(gen(3), 30, 8, 64, dtype=torch.bfloat16)
    for new, ctx in ((5, 300), (30, 310)):
        lens, cu, mask = i32([ctx]), i32([0, new]), words_of(ancestors(tree(random.Random(1), new)), 1)
        a, b = (paged.tree_attention(q[:new], c, table, lens, cu, mask, max_new=new) for c in (near, far))
        assert torch.equal(a, b)
        path = i32([[0, 2, 4]])
        a, b = (paged.compact([c], table, lens, cu, path, i32([3])) for c in (near, far))
        assert torch.equal(a, b) and torch.equal(near.k, far.k) and torch.equal(near.v, far.v)
    # rows 2^26 elements apart
    x = room.as_strided((36, 1000), (1 << 26, 1))
    x.copy_(randn(gen(4), 36, 1000, dtype=torch.bfloat16))
    tokens, parents, cu = i64(x.argmax(1).tolist()), i32([-1] + list(range(35))), i32([0, 36])
    for g, w in zip(paged.verify(x, tokens, parents, cu), paged.verify(x.contiguous(), tokens, parents, cu)):
        assert torch.equal(g, w)
    f8 = ops.F8Weight.from_float(randn(gen(5), 300, 1000, dtype=torch.bfloat16))
    for m in (36, 8):
        assert torch.equal(ops.linear_f8(x[36 - m:], f8), ops.linear_f8(x[36 - m:].contiguous(), f8))
    assert torch.equal(ops.linear_f8(x[::5], f8), ops.linear_f8(x[::5].contiguous(), f8))
    assert status() == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_captured_step_of_drafted_tokens(dtype):
    """Plan, append, tree attention, acceptance and move as one graph over two layers, replayed step after step without the host
    between them: the caches and lengths are those of the accepted tokens alone, fed one after another."""
    ops, paged = mods()
    g = gen(17)
    seqs, n, page, nh, nkv, hd, layers, vocab, width = 5, 12, 16, 4, 2, 64, 2, 40, 12
    pages = seqs * width
    caches = [paged.PagedCache(pages, page, nkv, hd, dtype) for _ in range(layers)]
    for c in caches:
        c.k.zero_(), c.v.zero_()
    # a model of one lookup: a token and its position decide q, k, v and the next token's logits
    table_qkv = randn(g, vocab, (nh + 2 * nkv) * hd, dtype=dtype)
    follows = randn(g, vocab, vocab, dtype=torch.float32)
    freq = 1.0 / 1e4 ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float32) / hd)
    table = torch.zeros(seqs, width, dtype=torch.int32, device="cuda")
    lens, held = i32([0] * seqs), i32([0] * seqs)
    free, count = torch.randperm(pages, device="cuda", generator=g).to(torch.int32), i32([pages])
    new, total = i32([n] * seqs), seqs * n
    tokens, parents = torch.zeros(total, dtype=torch.int64, device="cuda"), torch.zeros(total, dtype=torch.int32, device="cuda")
    blank = paged.plan(table.clone(), lens, new, page, total, held=held, free_pages=free, free_count=count, parents=parents, max_new=n)
    plan_out = blank._replace(held=held, free_count=count)

    def step():
        p = paged.plan(table, lens, new, page, total, held=held, free_pages=free, free_count=count, parents=parents, max_new=n, out=plan_out)
        qkv, outs = table_qkv[tokens], []
        for c in caches:
            q = paged.norm_rope_append(qkv, c, p.positions, p.slots, nh, freq)
            outs.append(paged.tree_attention(q, c, table, p.seq_lens, p.cu_new, p.mask, max_new=n))
        v = paged.verify(follows[tokens], tokens, parents, p.cu_new, max_new=n)
        paged.compact(caches, table, p.seq_lens, p.cu_new, v.path, v.accepted, out=lens)
        return outs, v

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs, v = step()
    rng = random.Random(9)
    best = follows.argmax(1).tolist()
    current, texts = [rng.randrange(vocab) for _ in range(seqs)], [[] for _ in range(seqs)]
    for _ in range(8):
        drafted, shape = [], []
        for s in range(seqs):
            tree_s = tree(rng, n)
            toks = [current[s]]
            for i in range(1, n):
                toks.append(best[toks[tree_s[i]]] if rng.random() < 0.7 else rng.randrange(vocab))
            drafted += toks
            shape += tree_s
        tokens.copy_(i64(drafted))
        parents.copy_(i32(shape))
        graph.replay()
        torch.cuda.synchronize()
        for s, (path, k) in enumerate(zip(v.path.tolist(), v.accepted.tolist())):
            texts[s] += [drafted[s * n + i] for i in path[:k]]
            assert all(b == best[a] for a, b in zip(texts[s], texts[s][1:]))
            current[s] = int(v.next[s])
        assert lens.tolist() == [len(t) for t in texts]
    assert max(lens.tolist()) > 12 and count.item() == pages - int(held.sum())
    # the same texts fed plainly
    for s, text in enumerate(texts):
        plain = paged.PagedCache(width, page, nkv, hd, dtype)
        t = i64(text)
        pos = torch.arange(len(text), device="cuda")
        q = paged.norm_rope_append(table_qkv[t], plain, pos, pos, nh, freq)
        for c in caches:
            at = table[s, pos // page].long()
            assert torch.equal(c.k[at, :, pos % page], plain.k[pos // page, :, pos % page])
            assert torch.equal(c.v[at, :, pos % page], plain.v[pos // page, :, pos % page])
    assert status() == 0


@gpu
def test_a_captured_step_that_runs_out_of_pages_keeps_what_it_refuses():
    """Plan, acceptance and move as one graph with lengths, pages held and the free count in place: sequences that find no pages, or no rows
    left, have the context they had, nothing is accepted for them, and they go on once there are pages."""
    _, paged = mods()
    rng = random.Random(3)
    seqs, n, page, width, vocab, rows = 6, 14, 16, 8, 30, 75   # (rows for five sequences and five tokens)
    cache = paged.PagedCache(64, page, 2, 64)
    cache.k.normal_(), cache.v.normal_()
    before, held = [5, 30, 0, 47, 17, 60], [1, 2, 0, 3, 2, 4]
    order = list(range(64))
    rng.shuffle(order)
    table = i32([[order.pop() for _ in range(h)] + [-1] * (width - h) for h in held])
    free, count, lens, held = i32(order), i32([3]), i32(before), i32(held)
    new, parents = i32([n] * seqs), i32([p for _ in range(seqs) for p in tree(rng, n)][:rows])
    logits, tokens = torch.empty(rows, vocab, device="cuda"), torch.empty(rows, dtype=torch.int64, device="cuda")
    args = dict(held=held, free_pages=free, free_count=count, parents=parents, max_new=n)
    out = paged.plan(table.clone(), lens, new, page, rows, **args)._replace(held=held, free_count=count)

    def step():
        p = paged.plan(table, lens, new, page, rows, out=out, **args)
        v = paged.verify(logits, tokens, parents, p.cu_new, max_new=n, seq_lens=p.seq_lens)
        paged.compact([cache], table, p.seq_lens, p.cu_new, v.path, v.accepted, out=lens)
        return v

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        v = step()
    refused = set()
    for turn in range(4):
        if turn == 2:
            count.fill_(40)   # others have given theirs back
        logits.normal_(generator=gen(turn))
        top, shape = logits.argmax(1).tolist(), parents.tolist()
        tokens.copy_(i64([top[at // n * n + shape[at]] if shape[at] >= 0 and rng.random() < 0.8 else 1 for at in range(rows)]))
        start, pages, left, was = lens.tolist(), held.tolist(), count.item(), table.tolist()
        want, _ = plain_plan(was, start, [n] * seqs, page, rows, pages, free.tolist(), left, shape, 1)
        path = plain_verify(logits, tokens.tolist(), shape, [n] * 5 + [5], n)
        graph.replay()
        torch.cuda.synchronize()
        for s in range(seqs):
            ok = want["seq_lens"][s] > 0
            assert v.accepted[s].item() == (path[0][s].item() if ok else 0) and v.next[s].item() == (path[2][s].item() if ok else -1)
            assert lens[s].item() == start[s] + v.accepted[s].item()
            refused |= set() if ok else {(turn, s)}
        assert held.tolist() == want["held"] and count.item() == want["free_count"][0]
    assert {s for t, s in refused if t < 2} > {5} and {s for t, s in refused if t >= 2} == {5} and status() == 0


# ------------------------------------------------------------------------------- refusals of the C ABI (no GPU)

def test_no_warp_of_the_kernels_meets_others_on_the_way():
    """As in the chunk kernels: every wait is bounded and a warp whose wait gave up leaves its loop, so no barrier among some of a
    CTA's warps stands there."""
    for name in ("lb_f8.cu", "lb_draft.cu"):
        source = (_lib.LIB_PATH.parent.parent / "csrc" / name).read_text()
        assert "named_barrier(" not in source and "bar.sync" not in source and "barrier.sync" not in source, name


def test_branches_that_all_lanes_have_to_take_alike_are_voted():
    """bra.uni promises that a warp's lanes agree, but each lane's wait answers for itself: the block that branches takes a vote first."""
    found = 0
    for path in sorted((_lib.LIB_PATH.parent.parent / "csrc").glob("*.cu*")):
        for block in re.findall(r"asm volatile\((.*?)\);", path.read_text(), re.S):
            if "bra.uni" in block:
                found += 1
                assert "vote.sync" in block[:block.index("bra.uni")], path.name
    assert found


def test_abi_refusals_of_what_lies_over_the_inputs_or_is_misaligned():
    lib = _lib.load_library()

    def cache(k, v):
        return _lib.PagedCacheStruct(k=k, v=v, k_page_stride=2048, v_page_stride=2048, num_pages=4, dtype=0, nkv=2, hd=64, page_size=16)

    def compact(caches, table=A, lens=A, cu=2 * A, path=3 * A, count=4 * A, out=5 * A, seqs=3, most=4):
        ptrs = (ctypes.c_void_p * len(caches))(*[ctypes.addressof(c) for c in caches])
        return lib.lb_paged_compact(ptrs, len(caches), table, 3, 3, lens, cu, path, count, seqs, most, out, 0, None)

    one = [cache(A, 2 * A)]
    for out in (A, A + 8, A - 8, 2 * A + 12, 2 * A - 8, 3 * A + 44, 4 * A + 4):
        assert compact(one, out=out) == 1 and "over an input" in message(lib), out
    for caches in ([cache(A, A)], one + [cache(3 * A, A)], [cache(i * A, (i + 40) * A) for i in range(1, 30)] + [cache(7 * A, 90 * A)]):
        assert compact(caches) == 1 and "twice" in message(lib)
    for kw in (dict(table=A + 2), dict(lens=A + 1), dict(cu=2 * A + 2), dict(path=A + 2), dict(count=A + 2), dict(out=5 * A + 2)):
        assert compact(one, **kw) == 2, kw

    def plan(lens=A, new=A, table=A, cu=A, pos=A, slots=A, parents=A, mask=A):
        return lib.lb_paged_plan(lens, new, 2, table, 4, 4, 16, 8, None, None, 0, None, parents, 1, cu, A, None, None, pos, slots, mask, None)

    for kw in (dict(lens=A + 2), dict(new=A + 1), dict(table=A + 2), dict(cu=A + 2), dict(pos=A + 4), dict(slots=A + 4), dict(parents=A + 2), dict(mask=A + 2)):
        assert plan(**kw) == 2, kw

    def verify(drafted=A, parents=A, cu=A, acc=A, path=A, after=A, targets=A):
        return lib.lb_draft_verify(A, 0, 100, 4, 100, drafted, parents, cu, 1, 4, 4, acc, path, after, targets, A, 1 << 30, None)

    for kw in (dict(drafted=A + 4), dict(parents=A + 2), dict(cu=A + 2), dict(acc=A + 2), dict(path=A + 2), dict(after=A + 4), dict(targets=A + 4)):
        assert verify(**kw) == 2, kw

    def linear(x, y, m=3, n=8, k=64, ldx=64):
        return lib.lb_f8_linear(x, 0, ldx, A, 64, A, None, y, m, n, k, A, 1 << 40, None)

    for x, y in ((A, A), (A, A + 2 * (2 * 64 + 63)), (A + 2 * 23, A)):
        assert linear(x, y) == 1 and "overlap" in message(lib), (x, y)


def test_compact_refuses_lengths_over_the_page_table():
    lib = _lib.load_library()
    cache = _lib.PagedCacheStruct(k=A, v=2 * A, k_page_stride=2048, v_page_stride=2048, num_pages=4, dtype=0, nkv=2, hd=64, page_size=16)
    ptrs = (ctypes.c_void_p * 1)(ctypes.addressof(cache))
    for out in (8 * A, 8 * A + 68, 8 * A - 8):   # three rows of four entries, seven apart
        assert lib.lb_paged_compact(ptrs, 1, 8 * A, 7, 4, A, 2 * A, 3 * A, 4 * A, 3, 4, out, 0, None) == 1 and "over an input" in message(lib), out


def test_f8_abi_refusals():
    lib = _lib.load_library()
    quant = lambda w=A, t=0, n=4, k=64, ldw=64, q=A, ldq=64, s=A: lib.lb_f8_quantize_weight(w, t, n, k, ldw, q, ldq, s, None)
    assert quant(w=None) == 1 and "null" in message(lib)
    for kw in (dict(t=3), dict(n=0), dict(k=0), dict(ldw=63), dict(ldq=72), dict(ldq=48), dict(k=131073, ldw=131073, ldq=131088), dict(n=65536 * 128)):
        assert quant(**kw) == 1, kw
    assert quant(w=MIS) == 2 and quant(q=MIS) == 2 and quant(s=A + 2) == 2 and quant(w=A + 2, t=2) == 2
    lin = lambda t=0, w=A, ldw=64, b=None, y=A, m=1, n=8, k=64, ws=A, wsb=1 << 40: lib.lb_f8_linear(A, t, k, w, ldw, A, b, y, m, n, k, ws, wsb, None)
    for kw in (dict(t=2), dict(w=None), dict(y=None), dict(n=0), dict(m=0), dict(m=65536 * 16), dict(k=131073, ldw=131088)):
        assert lin(**kw) == 1, kw
    assert lin(w=MIS) == 2 and lin(b=MIS) == 2 and lin(y=MIS) == 2
    assert lib.lb_f8_workspace(0, 8, 64) == 0
    need = lib.lb_f8_workspace(300, 8, 64)
    assert need > 0 and lin(m=300, wsb=need - 1) == 1 and "workspace" in message(lib)
    assert lin(m=300, ws=MIS) == 2


def test_draft_abi_refusals():
    lib = _lib.load_library()

    def plan(lens=A, seqs=2, table=A, stride=4, width=4, page=16, t=8, held=None, free=None, nf=0, count=None, parents=None, words=0, cu=A,
             held_out=None, count_out=None, pos=A, mask=None):
        return lib.lb_paged_plan(lens, A, seqs, table, stride, width, page, t, held, free, nf, count, parents, words, cu, A, held_out, count_out, pos, A,
                                 mask, None)

    for kw in (dict(lens=None), dict(table=None), dict(cu=None), dict(pos=None), dict(seqs=0), dict(seqs=8193), dict(stride=3), dict(width=0),
               dict(width=2 ** 28, stride=2 ** 28), dict(page=8), dict(page=40), dict(t=-1), dict(t=2 ** 30), dict(held=A), dict(held=A, free=A, count=A),
               dict(free=A, count=A), dict(parents=A), dict(mask=A), dict(parents=A, mask=A, words=0), dict(parents=A, mask=A, words=33),
               dict(held=A, free=A, count=A, held_out=A, count_out=A, nf=-1)):
        assert plan(**kw) == 1, kw

    def verify(x=A, t=0, ld=100, n=4, vocab=100, seqs=1, new=4, path=4, ws=A, wsb=1 << 30, acc=A):
        return lib.lb_draft_verify(x, t, ld, n, vocab, A, A, A, seqs, new, path, acc, A, A, A, ws, wsb, None)

    for kw in (dict(x=None), dict(t=3), dict(ld=99), dict(n=0), dict(n=2 ** 21), dict(vocab=0), dict(seqs=0), dict(new=0), dict(new=1025), dict(path=0),
               dict(path=1025), dict(acc=None), dict(ws=None), dict(wsb=0)):
        assert verify(**kw) == 1, kw
    assert verify(x=MIS) == 2 and verify(x=A + 2, t=2) == 2 and verify(ws=A + 8) == 2
    assert lib.lb_draft_verify_workspace(0, 100) == 0 and lib.lb_draft_verify_workspace(4, 100) == 32

    def cache(**kw):
        return _lib.PagedCacheStruct(**{**dict(k=A, v=A, k_page_stride=2 * 16 * 64, v_page_stride=2 * 16 * 64, num_pages=4, dtype=0, nkv=2, hd=64,
                                               page_size=16), **kw})

    def compact(caches, layers=None, table=A, stride=3, width=3, lens=A, seqs=1, path=4, out=2 * A):
        ptrs = (ctypes.c_void_p * max(1, len(caches)))(*[ctypes.addressof(c) for c in caches])
        return lib.lb_paged_compact(ptrs, len(caches) if layers is None else layers, table, stride, width, lens, A, A, A, seqs, path, out, 0, None)

    two = [cache(), cache()]
    for kw in (dict(layers=0), dict(layers=129), dict(table=None), dict(stride=2), dict(width=0), dict(seqs=0), dict(seqs=65536), dict(path=0), dict(path=1025),
               dict(out=A), dict(out=None)):
        assert compact(two, **kw) == 1, kw
    for other in (cache(dtype=1), cache(nkv=1), cache(num_pages=5), cache(k_page_stride=4096), cache(page_size=32, nkv=1), cache(k=None)):
        assert compact([cache(), other]) == 1
    ok = _lib.PagedCacheStruct(k=A, v=A, k_page_stride=2048, v_page_stride=2048, num_pages=4, dtype=0, nkv=2, hd=64, page_size=16)

    def tree_attention(mask=A, words=1, q=A):
        return lib.lb_paged_tree_attention(q, 256, 64, 4, 4, ctypes.addressof(ok), A, 3, 3, A, A, 2, mask, words, 1, 9, 0.1, A, 256, A, 1 << 40, None)

    assert tree_attention(mask=None) == 1 and tree_attention(words=0) == 1 and tree_attention(q=None) == 1
    assert tree_attention(mask=A + 2) == 2 and tree_attention(q=A + 8) == 2
