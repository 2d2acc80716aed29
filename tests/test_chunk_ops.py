"""The operators of a chunk of new tokens against plain implementations in 64 bits (B200 only, but for the refusals of
the C ABI, which come before any CUDA call).

Tolerances, with u = 2^-11 (fp16) or 2^-8 (bf16) the relative rounding of one stored value:
  * linear_w8: the quantized activations are fp32 products and one rint, reproduced here bit for bit, and the sum is
    exact, so y is the 64-bit value to u plus four fp32 roundings (2^-22 of |sum s t| + |bias|);
  * norm_rope_append: u plus 2^-18 of the pair's length (a sum of up to 256 squares, rsqrt, two products, cos and sin
    good to a few 2^-24 each);
  * attention: u of the result, and of A = sum p|v| / sum p: 1.25 u where the softmax weights are rounded to the
    type before the product with V, 2^-12 for exp2 and the fp32 sums of scores up to a few tens; for fp16 also
    L 2^-25 max|v|, the weights' absolute rounding below fp16's normal range.
Every tolerance adds 2^-24, half of fp16's smallest step, twice.
"""
import copy
import ctypes
import math
import pickle
import random

import pytest
import torch

from lowbit import _lib

gpu = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float16, torch.bfloat16]
TINY = 2.0 ** -23


def mods():
    from lowbit import ops, paged
    return ops, paged


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def close(got, want, tol, what=""):
    assert got.shape == want.shape
    bad = ~((got.double() - want).abs() <= tol + TINY)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {((got.double() - want).abs() / (tol + TINY)).max().item():.3g} of the tolerance"


# ------------------------------------------------------------------------------------------------------ linear_w8

def plain_quantize(x):
    x = x.float()
    amax = x.abs().amax(1, keepdim=True)
    # tensor / tensor: with a plain number on either side torch multiplies by a reciprocal, two roundings
    c = torch.full_like(amax, 127.0)
    r = torch.where(amax > 0, c / amax, torch.zeros_like(amax))
    return (x * r).round().clamp(-127, 127), (amax / c)[:, 0]


def check_linear(x, q, s, bias, y):
    qx, sx = plain_quantize(x)
    prod = (qx.double() @ q.double().t()) * sx.double()[:, None] * s.double()
    want = prod if bias is None else prod + bias.double()
    mag = prod.abs() if bias is None else prod.abs() + bias.double().abs()
    close(y, want, U[y.dtype] * want.abs() + 2.0 ** -22 * mag, f"M={x.shape[0]} K={x.shape[1]} N={q.shape[0]}")


ROWS = [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 100, 128, 129, 255, 256, 257, 300, 513]
WIDTHS = [(16, 1), (1, 5), (100, 37), (128, 128), (129, 130), (384, 1001), (896, 128), (2048, 256), (1000, 2000), (4864, 896)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", WIDTHS)
def test_linear_w8(dtype, k, n):
    ops, _ = mods()
    g = gen(k * 7 + n)
    w = randn(g, n, k, std=0.05)
    w8 = ops.W8Weight.from_float(w)
    bias = randn(g, n, dtype=dtype)
    for m in ROWS:
        x = randn(g, m, k, dtype=dtype, std=2.0)
        x[m // 2] *= 0 if m > 3 else 1
        check_linear(x, w8.q, w8.scales, None, ops.linear_w8(x, w8))
        check_linear(x, w8.q, w8.scales, bias, ops.linear_w8(x, w8, bias=bias))
    assert ops.ext().lib.lb_device_error() == 0


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 16), (5, 33), (17, 128), (4, 1000), (2, 18944), (300, 896)])
def test_quantize_w8_is_the_formula_bit_for_bit(dtype, n, k):
    ops, _ = mods()
    w = randn(gen(n + k), n, k, dtype=dtype)
    w[0, 0] = 0
    if n > 2:
        w[1] = 0
        w[2] = w[2] * 1e-4
    q, s = ops.quantize_w8_gpu(w)
    want_q, want_s = plain_quantize(w)
    assert q.shape == (n, k) and torch.equal(q.float(), want_q) and torch.equal(s, want_s)


@gpu
def test_quantize_rows_of_subnormals_and_of_the_largest_values():
    ops, _ = mods()
    for dtype, least, most in ((torch.float16, 2.0 ** -24, 65504.0), (torch.bfloat16, 2.0 ** -133, 3.3895e38)):
        w = torch.tensor([[least, -2 * least, 4 * least], [most, -most / 4, most / 8]], device="cuda", dtype=dtype)
        q, s = ops.quantize_w8_gpu(w)
        assert q.tolist() == [[32, -64, 127], [127, -32, 16]]
        assert torch.allclose(s.double() * 127, w.double().abs().amax(1), rtol=1e-2)


@gpu
def test_linear_w8_rows_that_are_not_finite_stay_alone():
    ops, _ = mods()
    g = gen(5)
    w8 = ops.W8Weight.from_float(randn(g, 96, 256))
    for m in (4, 40, 200):
        x = randn(g, m, 256, dtype=torch.float16)
        clean = ops.linear_w8(x, w8)
        x[1, 3], x[2, 250] = float("nan"), float("inf")
        y = ops.linear_w8(x, w8)
        assert not torch.isfinite(y[1:3]).any()
        keep = [i for i in range(m) if i not in (1, 2)]
        assert torch.equal(y[keep], clean[keep])


@gpu
def test_linear_w8_extreme_sums_are_exact():
    """All-largest products: the int32 sum at K = 131072 is 127^2 * 131072 = 2114060288, just below 2^31."""
    ops, _ = mods()
    k = 131072
    q = torch.full((3, k), 127, device="cuda", dtype=torch.int8)
    q[1] = -127
    q[2, ::2] = -127
    w8 = ops.W8Weight(q, torch.full((3,), 2.0 ** -20, device="cuda"))
    for m in (1, 20, 130):
        y = ops.linear_w8(torch.ones(m, k, device="cuda", dtype=torch.float16), w8)
        want = torch.tensor([127.0 * k / 2 ** 20, -127.0 * k / 2 ** 20, 0.0], device="cuda").half()
        assert torch.equal(y, want.expand(m, 3))
    with pytest.raises(ValueError):
        ops.W8Weight(torch.zeros(1, k + 1, device="cuda", dtype=torch.int8), torch.ones(1, device="cuda"))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(100, 2500), (513, 4700), (2048, 4736), (5120, 2369), (9000, 2400), (10256, 2384)])
def test_linear_w8_up_to_forty_rows(dtype, k, n):
    ops, _ = mods()
    g = gen(k + n)
    w8 = ops.W8Weight.from_float(randn(g, n, k, std=0.05))
    bias = randn(g, n, dtype=dtype)
    for m in (1, 3, 8, 9, 16, 17, 24, 25, 40, 41):
        x = randn(g, m, k, dtype=dtype)
        check_linear(x, w8.q, w8.scales, bias, ops.linear_w8(x, w8, bias=bias))


@gpu
@pytest.mark.parametrize("k", [8193, 20000, 50001, 100000])
def test_linear_w8_long_rows(k):
    """Rows longer than the registers hold, and than shared memory holds; aligned to 16 bytes or to 2."""
    ops, _ = mods()
    g = gen(k)
    w8 = ops.W8Weight.from_float(randn(g, 70, k, std=0.05))
    for m in (3, 70):
        wide = randn(g, m, k + 9, dtype=torch.bfloat16)
        for off in (0, 1):
            x = wide[:, off:off + k]
            check_linear(x, w8.q, w8.scales, None, ops.linear_w8(x, w8))


@gpu
@pytest.mark.parametrize("m", [1, 8, 40])
def test_linear_w8_reads_weights_that_the_kernel_before_it_wrote(m):
    """Weights quantized into one pair of buffers again and again, each followed at once by a product: by default no
    weight is read before the kernel before it is done."""
    from lowbit._lib import DTYPE_IDS
    ops, _ = mods()
    g, n, k = gen(m), 256, 8192
    floats = [randn(g, n, k, std=0.01 * (i + 1)) for i in range(8)]
    w8 = ops.W8Weight.from_float(floats[0])
    x = randn(g, m, k, dtype=torch.float16)
    want = [ops.linear_w8(x, ops.W8Weight.from_float(f)) for f in floats]
    torch.cuda.synchronize()
    got = []
    for f in floats:
        rc = ops.ext().lib.lb_w8_quantize_rows(f.data_ptr(), DTYPE_IDS[f.dtype], n, k, k, w8.q.data_ptr(), k,
                                               w8.scales.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        got.append(ops.linear_w8(x, w8))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_linear_w8_strided_inputs_out_and_streams():
    ops, _ = mods()
    g = gen(11)
    w8 = ops.W8Weight.from_float(randn(g, 200, 320))
    wide = randn(g, 50, 700, dtype=torch.bfloat16)
    for m in (1, 13, 50):
        for off in (0, 3, 8):   # rows 700 elements apart, aligned to 16 bytes or not at all
            x = wide[:m, off:off + 320]
            out = torch.full((m, 200), float("nan"), device="cuda", dtype=torch.bfloat16)
            y = ops.linear_w8(x, w8, out=out)
            assert y.data_ptr() == out.data_ptr()
            check_linear(x, w8.q, w8.scales, None, y)
            check_linear(x, w8.q, w8.scales, None, ops.linear_w8(x.t().contiguous().t(), w8))   # inner stride not 1
    side = torch.cuda.Stream()
    x = randn(g, 40, 320, dtype=torch.float16)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = ops.linear_w8(x, w8)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, ops.linear_w8(x, w8))
    assert ops.linear_w8(x[:0], w8).shape == (0, 200)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(629, 7531, 384), (2137, 6249, 1000), (2200, 9000, 500), (2200, 9001, 500), (1552, 11256, 3000),
                                   (1144, 15727, 3000), (973, 15400, 4096)])
def test_linear_w8_several_tiles_a_cta(dtype, m, n, k):
    """Large products: single CTAs with two and three tiles each, pairs with five, and pairs whose tiles are more than
    256 tokens wide, with two and three each; the last tile partial both ways, rows of 16-byte multiples and not."""
    ops, _ = mods()
    g = gen(m + n)
    w8 = ops.W8Weight.from_float(randn(g, n, k, std=0.05))
    bias = randn(g, n, dtype=dtype)
    x = randn(g, m, k, dtype=dtype, std=2.0)
    y = ops.linear_w8(x, w8, bias=bias)
    check_linear(x, w8.q, w8.scales, bias, y)
    assert torch.equal(y, ops.linear_w8(x, w8, bias=bias))
    assert ops.ext().lib.lb_device_error() == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_chunk_operators_give_the_same_bits_under_every_launch_option(dtype):
    """Programmatic launch off and on, static weights read before the wait and not: each operator several times in a row,
    over products of every kernel."""
    ops, paged = mods()
    e = ops.ext()
    g = gen(31)
    shapes = [(1, 2048, 512), (8, 512, 1536), (16, 1024, 4096), (40, 2048, 2048), (100, 896, 1536), (700, 2500, 1000)]
    weights = [(randn(g, m, k, dtype=dtype), ops.W8Weight.from_float(randn(g, n, k, std=0.05)), randn(g, n, dtype=dtype))
               for m, n, k in shapes]
    nh, nkv, hd = 14, 2, 64
    norms = [(1 + randn(g, hd, std=0.1)).to(dtype) for _ in range(2)]
    freq = 1.0 / 1e6 ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float32) / hd)

    def once():
        out = [ops.linear_w8(x, w8, bias=b) for _ in range(3) for x, w8, b in weights]
        for new, ctx in (([1, 1], [300, 70]), ([40, 5], [300, 70])):
            q, cache, table, lens, cu = build(gen(32), new, ctx, nh, nkv, hd, 16, dtype, poison=False)
            pos = torch.cat([torch.arange(c - n, c, device="cuda") for n, c in zip(new, ctx)])
            seq = torch.repeat_interleave(torch.arange(2, device="cuda"), torch.tensor(new, device="cuda"))
            slots = table[seq, pos // 16].long() * 16 + pos % 16
            qkv = randn(gen(33), sum(new), (nh + 2 * nkv) * hd, dtype=dtype)
            q = paged.norm_rope_append(qkv, cache, pos, slots, nh, freq, *norms)
            out += [q, cache.k, cache.v, paged.attention(q, cache, table, lens, cu, max_new=max(new))]
        return out

    prev = {o: e.get_option(o) for o in ("pdl", "early_weights")}
    try:
        runs = []
        for pdl, early in ((0, 0), (1, 0), (1, 1)):
            e.set_option("pdl", pdl)
            e.set_option("early_weights", early)
            torch.cuda.synchronize()   # what wrote the weights is done
            runs.append(once())
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
    finally:
        torch.cuda.synchronize()
        for o, v in prev.items():
            e.set_option(o, v)
    assert e.lib.lb_device_error() == 0


@gpu
@pytest.mark.parametrize("k", [64, 100])
def test_a_copy_of_a_w8_weight_is_its_own(k):
    """copy.deepcopy and pickle: the copy multiplies with its own integers and scales, whatever becomes of the first."""
    ops, _ = mods()
    g = gen(k)
    for m in (3, 70):
        w8 = ops.W8Weight.from_float(randn(g, 48, k))
        x = randn(g, m, k, dtype=torch.float16)
        want = ops.linear_w8(x, w8)
        for other in (copy.deepcopy(w8), pickle.loads(pickle.dumps(w8)), copy.copy(w8)):
            assert torch.equal(ops.linear_w8(x, other), want)
        twin = copy.deepcopy(w8)
        w8.q.zero_(), w8.scales.zero_()
        assert torch.equal(ops.linear_w8(x, twin), want) and not ops.linear_w8(x, w8).any()
    for name in ("q", "scales"):
        with pytest.raises(AttributeError):
            setattr(w8, name, getattr(twin, name))


@gpu
def test_linear_w8_refusals():
    ops, _ = mods()
    w8 = ops.W8Weight.from_float(torch.randn(8, 64, device="cuda"))
    x = torch.zeros(2, 64, device="cuda", dtype=torch.float16)
    for bad in (x.float(), x[:, :32], x[0], x.cpu()):
        with pytest.raises(RuntimeError):
            ops.linear_w8(bad, w8)
    for kw in (dict(bias=torch.zeros(7, device="cuda", dtype=torch.float16)), dict(bias=torch.zeros(8, device="cuda")),
               dict(out=torch.zeros(2, 9, device="cuda", dtype=torch.float16)),
               dict(out=torch.zeros(8, 2, device="cuda", dtype=torch.float16).t())):
        with pytest.raises(RuntimeError):
            ops.linear_w8(x, w8, **kw)
    with pytest.raises(RuntimeError):
        ops.W8Weight(torch.zeros(4, 16, device="cuda"), torch.zeros(4, device="cuda"))
    with pytest.raises(RuntimeError):
        ops.W8Weight(torch.zeros(4, 16, device="cuda", dtype=torch.int8), torch.zeros(3, device="cuda"))


# ----------------------------------------------------------------------------------------------- norm_rope_append

def plain_append(qkv, nh, nkv, hd, pos, inv_freq, q_norm, k_norm, eps):
    x = qkv.double().view(qkv.shape[0], nh + 2 * nkv, hd)
    f = inv_freq.numel()
    angle = (pos.double()[:, None] * inv_freq.double())[:, None]
    parts, mags = [], []
    for h, w in ((x[:, :nh], q_norm), (x[:, nh:nh + nkv], k_norm)):
        if w is not None:
            h = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()
        a, b = h[..., :f], h[..., f:2 * f]
        parts.append(torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), h[..., 2 * f:]), -1))
        mag = torch.sqrt(a.square() + b.square())
        mags.append(torch.cat((mag, mag, h[..., 2 * f:].abs()), -1))
    return parts[0], parts[1], x[:, nh + nkv:], mags


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,hd,rot", [(16, 2, 128, 128), (14, 2, 64, 64), (4, 4, 80, 80), (3, 1, 256, 64), (8, 2, 96, 96),
                                           (5, 5, 16, 16), (7, 1, 128, 32), (2, 1, 64, 0), (130, 3, 128, 128)])
@pytest.mark.parametrize("norm", [False, True])
def test_norm_rope_append(dtype, nh, nkv, hd, rot, norm):
    ops, paged = mods()
    g = gen(nh * 100 + hd)
    inv_freq = 1.0 / 1e6 ** (torch.arange(0, rot, 2, device="cuda", dtype=torch.float32) / max(rot, 1))
    for t, page in ((1, 16), (3, 48), (41, 64)):
        width = (nh + 2 * nkv) * hd
        wide = randn(g, t, width + 24, dtype=dtype, std=1.5)
        qkv = wide[:, 8:8 + width]
        qn, kn = (1 + randn(g, hd, std=0.1)).to(dtype) if norm else None, (1 + randn(g, hd, std=0.1)).to(dtype) if norm else None
        pos = torch.randint(0, 500000, (t,), device="cuda", generator=g)
        pos[0] = 0
        pages = 5
        slots = torch.randperm(pages * page, device="cuda", generator=g)[:t].contiguous()
        if t > 3:
            slots[2] = -1
        both = randn(g, pages, 2, nkv, page, hd, dtype=dtype)
        before = both.clone()
        cache = paged.PagedCache.from_tensors(both[:, 0], both[:, 1])
        q = paged.norm_rope_append(qkv, cache, pos, slots, nh, inv_freq, q_norm=qn, k_norm=kn, eps=1e-5)
        wq, wk, wv, mags = plain_append(qkv, nh, nkv, hd, pos, inv_freq, qn, kn, 1e-5)
        tol = lambda w, m: U[dtype] * w.abs() + 2.0 ** -18 * m
        close(q, wq, tol(wq, mags[0]), "q")
        keep = slots >= 0
        at, row = (slots // page)[keep], (slots % page)[keep]
        close(cache.k[at, :, row], wk[keep], tol(wk, mags[1])[keep], "k")
        assert torch.equal(cache.v[at, :, row].double(), wv[keep])
        untouched = torch.ones(pages, page, dtype=torch.bool, device="cuda")
        untouched[at, row] = False
        assert torch.equal(both.permute(0, 3, 1, 2, 4)[untouched], before.permute(0, 3, 1, 2, 4)[untouched])
    assert ops.ext().lib.lb_device_error() == 0


@gpu
def test_append_slot_outside_the_cache_is_reported_and_not_written():
    ops, paged = mods()
    lib = ops.ext().lib
    cache = paged.PagedCache.from_tensors(*torch.zeros(2, 2, 1, 16, 64, device="cuda", dtype=torch.float16))
    qkv = torch.ones(2, 4 * 64, device="cuda", dtype=torch.float16)
    freq = torch.ones(32, device="cuda")
    paged.norm_rope_append(qkv, cache, torch.zeros(2, device="cuda", dtype=torch.int64),
                           torch.tensor([32, 5], device="cuda"), 2, freq)
    try:
        assert lib.lb_device_error() == 3
    finally:
        lib.lb_clear_device_error()
    assert lib.lb_device_error() == 0
    assert cache.v.float().sum().item() == 64 and cache.v[0, 0, 5].float().sum().item() == 64


@gpu
def test_append_refusals():
    _, paged = mods()
    cache = paged.PagedCache(2, 16, 1, 64)
    qkv = torch.zeros(2, 4 * 64, device="cuda", dtype=torch.float16)
    pos = torch.zeros(2, device="cuda", dtype=torch.int64)
    freq = torch.ones(32, device="cuda")
    ok = dict(qkv=qkv, cache=cache, positions=pos, slots=pos, nh=2, inv_freq=freq)
    norm = torch.ones(64, device="cuda", dtype=torch.float16)
    for kw in (dict(qkv=qkv.bfloat16()), dict(qkv=qkv[:, :192]), dict(qkv=qkv.cpu()), dict(nh=3), dict(nh=0),
               dict(positions=pos.int()), dict(slots=pos[:1]), dict(inv_freq=freq[:12]), dict(inv_freq=freq.double()),
               dict(inv_freq=torch.ones(40, device="cuda")), dict(q_norm=norm), dict(q_norm=norm, k_norm=norm[:32]),
               dict(out=torch.zeros(2, 3, 64, device="cuda", dtype=torch.float16))):
        with pytest.raises(RuntimeError):
            paged.norm_rope_append(**{**ok, **kw})
    with pytest.raises(ValueError):
        paged.PagedCache(2, 20, 1, 64)
    with pytest.raises(ValueError):
        paged.PagedCache(2, 16, 1, 72)
    with pytest.raises(RuntimeError):
        paged.PagedCache.from_tensors(torch.zeros(2, 1, 16, 64, device="cuda"), torch.zeros(2, 1, 16, 64, device="cuda"))


# ------------------------------------------------------------------------------------------------------ attention

def build(g, new, ctx, nh, nkv, hd, page, dtype, spare=2, std=1.5, poison=True):
    """A cache whose every row outside the contexts is NaN or infinite, and a table whose unused entries are garbage."""
    _, paged = mods()
    need = [-(-c // page) for c in ctx]
    pages, width = sum(need) + spare, max(need + [1]) + 1
    both = randn(g, pages, 2, nkv, page, hd, dtype=dtype)
    order = torch.randperm(pages, device="cuda", generator=g).tolist()
    table = torch.full((len(ctx), width), -7, dtype=torch.int32)
    table[:, ::2] = 2 ** 31 - 1
    live = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for s, (c, n) in enumerate(zip(ctx, need)):
        table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        for j in range(n):
            live[order[at + j], :min(page, c - j * page)] = True
        at += n
    if poison:
        dead = ~live.cuda()
        rows = both.permute(0, 3, 1, 2, 4)
        junk = torch.where(torch.rand(rows[dead].shape, device="cuda", generator=g) < 0.5, float("nan"), float("inf"))
        rows[dead] = junk.to(dtype)
    q = randn(g, sum(new), nh, hd, dtype=dtype, std=std)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    return (q, paged.PagedCache.from_tensors(both[:, 0], both[:, 1]), table.cuda(),
            torch.tensor(ctx, dtype=torch.int32, device="cuda"), cu)


def plain_attention(q, cache, table, ctx, new, scale):
    nh, hd = q.shape[1:]
    grp = nh // cache.nkv
    out, absv, top, t = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64), 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        if n and c:
            pages = table[s, : -(-c // cache.page_size)].long()
            k, v = (x[pages].permute(0, 2, 1, 3).reshape(-1, cache.nkv, hd)[:c].double().repeat_interleave(grp, 1)
                    for x in (cache.k, cache.v))
            score = torch.einsum("nhd,khd->hnk", q[t:t + n].double(), k) * scale
            last = c - n + torch.arange(n, device="cuda")
            score.masked_fill_(torch.arange(c, device="cuda") > last[:, None], float("-inf"))
            p = torch.nan_to_num(torch.softmax(score, -1), nan=0.0)
            out[t:t + n] = torch.einsum("hnk,khd->nhd", p, v)
            absv[t:t + n] = torch.einsum("hnk,khd->nhd", p, v.abs())
            top[t:t + n] = c * 2.0 ** -25 * v.abs().amax()
        t += n
    return out, absv, top


def check_attention(q, cache, table, ctx, new, y, scale):
    want, absv, top = plain_attention(q, cache, table, ctx, new, scale)
    u = U[q.dtype]
    tol = u * want.abs() + (1.25 * u + 2.0 ** -12) * absv + (top if q.dtype == torch.float16 else 0)
    close(y, want, tol, f"new={new[:4]} ctx={ctx[:4]}")
    blind = want.abs().amax((1, 2)) == 0
    assert (y[blind] == 0).all()


def run_attention(g, new, ctx, nh, nkv, hd, page, dtype, **kw):
    ops, paged = mods()
    q, cache, table, lens, cu = build(g, new, ctx, nh, nkv, hd, page, dtype)
    y = paged.attention(q, cache, table, lens, cu, **kw)
    check_attention(q, cache, table, ctx, new, y, kw.get("scale") or 1 / math.sqrt(hd))
    again = paged.attention(q, cache, table, lens, cu, **kw)
    assert torch.equal(y, again)   # the same bits every time
    assert ops.ext().lib.lb_device_error() == 0


HEADS = [(16, 2, 128), (28, 4, 128), (14, 2, 64), (12, 2, 128), (4, 4, 64), (9, 1, 128), (16, 1, 64), (40, 1, 128), (1, 1, 128)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_attention_single_tokens(dtype, nh, nkv, hd):
    g = gen(nh + hd)
    for page in (16, 48, 128):
        for ctx in ([1], [15], [16], [17], [127, 128, 129, 0, 1], [1000, 2, 513], [5000]):
            run_attention(g, [1] * len(ctx), ctx, nh, nkv, hd, page, dtype, max_new=1)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_attention_chunks(dtype, nh, nkv, hd):
    g = gen(2 * nh + hd)
    for page, new, ctx in ((16, [1], [1]), (16, [2], [2]), (32, [3, 5], [70, 5]), (64, [17], [64]), (48, [40], [300]),
                           (256, [64, 1, 0, 130], [64, 77, 20, 700]), (128, [129], [129]), (16, [300], [1111]),
                           (80, [257, 2, 33], [600, 1500, 33])):
        run_attention(g, new, ctx, nh, nkv, hd, page, dtype)
        if max(new) > 1:
            run_attention(g, new, ctx, nh, nkv, hd, page, dtype, max_new=max(new), max_len=max(ctx))


@gpu
@pytest.mark.parametrize("new,ctx", [([5], [3]), ([40, 3], [7, 0]), ([1, 1, 1], [0, 0, 4]), ([0, 0], [9, 0]), ([200], [130])])
def test_attention_rows_without_keys_are_zero(new, ctx):
    """Contexts shorter than the new tokens: the first ones see no key; sequences without tokens or without context."""
    if sum(new) == 0:
        new = new + [1]
        ctx = ctx + [1]
    for hd, nh, nkv in ((64, 6, 2), (128, 16, 2), (128, 40, 1)):
        for dtype in DTYPES:
            run_attention(gen(sum(ctx)), new, ctx, nh, nkv, hd, 16, dtype)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,ctx", [(1, 300), (2, 40), (100, 300), (300, 1500)])
def test_attention_scores_that_are_not_finite_reach_the_rows_that_see_them(dtype, new, ctx):
    """A key of NaN, or one that gives an infinite score: every row that sees it is NaN, as exp(inf - inf) is, and the
    rows before it are untouched. Keys at every place of a block, since the exponentials are not all taken the same way."""
    ops, paged = mods()
    q, cache, table, lens, cu = build(gen(6), [new], [ctx], 16, 2, 128, 32, dtype)
    q = q.abs()
    clean = paged.attention(q, cache, table, lens, cu, max_new=new)
    for back in {1, 2, 3, 5, 8, 12, 17, new // 2, new}:
        key = ctx - back
        at, row = int(table[0, key // 32]), key % 32
        keep = cache.k[at, :, row].clone()
        for bad in (float("nan"), float("inf")):
            cache.k[at, :, row] = bad
            y = paged.attention(q, cache, table, lens, cu, max_new=new)
            first = max(0, new - back)   # the first new token that sees the key
            assert torch.isnan(y[first:]).all(), (back, bad)
            assert torch.equal(y[:first], clean[:first]), (back, bad)
        cache.k[at, :, row] = keep


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,ctx", [(2, 40), (100, 300), (300, 1500)])
def test_attention_values_of_unseen_keys_have_no_weight(dtype, hd, new, ctx):
    """Values at the end of the type's range: rows before the key are bit for bit what they were. Keys at every place of
    a block, since the exponentials are not all taken the same way."""
    _, paged = mods()
    q, cache, table, lens, cu = build(gen(16), [new], [ctx], 16, 2, hd, 32, dtype)
    clean = paged.attention(q, cache, table, lens, cu, max_new=new)
    for back in sorted({b for b in (*range(1, 18), new // 2) if b < new}):
        key = ctx - back
        at, row = int(table[0, key // 32]), key % 32
        keep = cache.v[at, :, row].clone()
        cache.v[at, :, row] = -0.9 * torch.finfo(dtype).max
        y = paged.attention(q, cache, table, lens, cu, max_new=new)
        assert torch.equal(y[:new - back], clean[:new - back]), back
        cache.v[at, :, row] = keep


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_large_scores_and_constant_rows(dtype):
    """Scores far apart (one key takes all the weight; the maximum found first, or last) and all alike."""
    ops, paged = mods()
    g = gen(3)
    for new, ctx in (([1], [700]), ([150], [700])):
        q, cache, table, lens, cu = build(g, new, ctx, 16, 2, 128, 32, dtype)
        first, last = int(table[0, 0]), int(table[0, 20])
        for page in (first, last):
            cache.k[page, :, 3] = 8.0
            qq = q.abs()
            y = paged.attention(qq, cache, table, lens, cu, max_new=max(new))
            check_attention(qq, cache, table, ctx, new, y, 1 / math.sqrt(128))
        zero = torch.zeros_like(q)
        check_attention(zero, cache, table, ctx, new, paged.attention(zero, cache, table, lens, cu, max_new=max(new)), 1 / math.sqrt(128))
        y = paged.attention(q, cache, table, lens, cu, max_new=max(new), scale=0.5)
        check_attention(q, cache, table, ctx, new, y, 0.5)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(28, 4, 128), (16, 2, 128), (14, 2, 64), (8, 8, 64)])
def test_attention_many_ragged_sequences(dtype, nh, nkv, hd):
    """More sequences than a warp has lanes, of long and empty contexts, more row tiles than SMs, and dozens of key tiles
    one after another in a CTA."""
    rng = random.Random(nh + hd)
    for seqs, most_new, most_ctx in ((33, 60, 700), (70, 90, 5000)):
        new = [rng.choice((0, 1, rng.randint(1, most_new), most_new)) for _ in range(seqs)]
        new[seqs // 2] = most_new
        ctx = [rng.choice((0, n, n + rng.randint(0, most_ctx), most_ctx)) for n in new]
        ctx[0] = most_ctx
        run_attention(gen(seqs), new, ctx, nh, nkv, hd, 48, dtype, max_new=most_new)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(28, 4, 128), (14, 2, 64)])
def test_attention_long_chunk(dtype, nh, nkv, hd):
    """Row tiles for every SM over a long context, which no cluster splits: 95 key tiles in each CTA's ring."""
    run_attention(gen(hd), [2700], [12150], nh, nkv, hd, 64, dtype)


@gpu
def test_attention_strides_streams_and_graph():
    """q as a slice of the fused projection's rows, a table that is a slice of a wider one, another stream, a captured
    graph replayed over new lengths, and tokens behind the last sequence left unwritten."""
    ops, paged = mods()
    g = gen(8)
    for new, ctx in (([1, 1, 1], [200, 31, 640]), ([60, 1, 7], [200, 31, 640])):
        q, cache, table, lens, cu = build(g, new, ctx, 8, 2, 64, 32, torch.float16)
        t = q.shape[0]
        fused = torch.zeros(t, 20, 64, device="cuda", dtype=torch.float16)
        fused[:, 1:17:2] = q
        wide = torch.full((3, table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table
        want = paged.attention(q, cache, table, lens, cu, max_new=max(new))
        got = paged.attention(fused[:, 1:17:2], cache, wide[:, :table.shape[1]], lens, cu, max_new=max(new))
        assert torch.equal(want, got)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        out = torch.full((t + 2, 8, 64), 7.0, device="cuda", dtype=torch.float16)
        padded = torch.cat((q, q[:2]))
        with torch.cuda.stream(side):
            paged.attention(padded, cache, table, lens, cu, max_new=max(new), out=out)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out[:t], want) and (out[t:] == 7).all()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = paged.attention(q, cache, table, lens, cu, max_new=max(new))
        shorter = [c - 20 if c > 100 else c for c in ctx]
        lens.copy_(torch.tensor(shorter, dtype=torch.int32))
        graph.replay()
        check_attention(q, cache, table, shorter, new, y, 0.125)


@gpu
def test_attention_and_append_past_2_to_31_elements():
    """A cache of 2.2e9 values: the last pages' offsets do not fit 32 bits."""
    ops, paged = mods()
    nkv, page, hd = 4, 256, 128
    pages = (2 ** 31 + 2 ** 26) // (nkv * page * hd)
    k = torch.empty(pages, nkv, page, hd, device="cuda", dtype=torch.float16)
    v = torch.empty_like(k)
    g = gen(21)
    k[-3:] = randn(g, 3, nkv, page, hd, dtype=torch.float16)
    v[-3:] = randn(g, 3, nkv, page, hd, dtype=torch.float16)
    cache = paged.PagedCache.from_tensors(k, v)
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32, device="cuda")
    for new in (1, 90):
        ctx = 600
        pos = torch.arange(ctx - new, ctx, device="cuda")
        qkv = randn(g, new, (8 + 8) * hd, dtype=torch.float16)
        slots = table[0].long()[pos // page] * page + pos % page
        freq = 1.0 / 1e6 ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float32) / hd)
        q = paged.norm_rope_append(qkv, cache, pos, slots, 8, freq)
        assert torch.equal(v[slots // page, :, slots % page].reshape(new, -1), qkv[:, 12 * hd:])
        y = paged.attention(q, cache, table, torch.tensor([ctx], dtype=torch.int32, device="cuda"),
                            torch.tensor([0, new], dtype=torch.int32, device="cuda"), max_new=new)
        check_attention(q, cache, table, [ctx], [new], y, 1 / math.sqrt(hd))
    assert ops.ext().lib.lb_device_error() == 0


@gpu
@pytest.mark.parametrize("new", [1, 100])
def test_attention_reports_a_page_outside_the_cache(new):
    ops, paged = mods()
    lib = ops.ext().lib
    q, cache, table, lens, cu = build(gen(4), [new], [200], 4, 2, 64, 16, torch.float16, poison=False)
    table[0, 3] = cache.num_pages
    y = paged.attention(q, cache, table, lens, cu, max_new=new)
    try:
        assert lib.lb_device_error() == 3
        assert torch.isfinite(y).all()
    finally:
        lib.lb_clear_device_error()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 5, 100])
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 48), (128, 128)])
def test_attention_keys_of_a_page_outside_the_cache_count_as_zeros(dtype, new, hd, page):
    """Entries below and above the cache, in the middle and at the end of a context: the same as a page of zeros; no other
    page, the first one above all, takes their place."""
    ops, paged = mods()
    lib = ops.ext().lib
    q, cache, table, lens, cu = build(gen(14), [new], [700], 8, 2, hd, page, dtype, spare=3)
    swap = table == 0   # no context holds page 0: the last spare page takes its place
    spare = next(i for i in range(1, cache.num_pages) if not (table[0, :-(-700 // page)] == i).any())
    cache.k[spare], cache.v[spare] = cache.k[0].clone(), cache.v[0].clone()
    table[swap] = spare
    cache.k[0], cache.v[0] = 3.0, float("nan")
    last = -(-700 // page) - 1
    table[0, 1], table[0, 3], table[0, last - 1], table[0, last] = -1, cache.num_pages, -2 ** 31, 2 ** 31 - 1
    y = paged.attention(q, cache, table, lens, cu, max_new=new)
    assert lib.lb_device_error() == 3
    lib.lb_clear_device_error()
    whole = paged.PagedCache.from_tensors(*(torch.cat((x, torch.zeros_like(x[:1]))) for x in (cache.k, cache.v)))
    zeros = table.clone()
    zeros[0, [1, 3, last - 1, last]] = cache.num_pages
    check_attention(q, whole, zeros, [700], [new], y, 1 / math.sqrt(hd))
    assert torch.equal(y, paged.attention(q, whole, zeros, lens, cu, max_new=new))
    assert lib.lb_device_error() == 0


@gpu
def test_attention_refusals():
    _, paged = mods()
    q, cache, table, lens, cu = build(gen(4), [2, 1], [20, 9], 4, 2, 64, 16, torch.float16)
    ok = dict(q=q, cache=cache, page_table=table, seq_lens=lens, cu_new=cu)
    for kw in (dict(q=q.bfloat16()), dict(q=q[..., :32]), dict(q=q[:, :3]), dict(q=q.cpu()), dict(q=q[0]),
               dict(page_table=table.long()), dict(page_table=table[0]), dict(page_table=table[:1]),
               dict(seq_lens=lens.long()), dict(seq_lens=lens[:1]), dict(cu_new=cu[:2]), dict(max_new=0), dict(max_len=0),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(out=torch.zeros(3, 4, 32, device="cuda", dtype=torch.float16))):
        with pytest.raises(RuntimeError):
            paged.attention(**{**ok, **kw})
    big = paged.PagedCache(2, 16, 1, 96)
    with pytest.raises(RuntimeError, match="64 and 128"):
        paged.attention(torch.zeros(3, 2, 96, device="cuda", dtype=torch.float16), big, table, lens, cu)


# ------------------------------------------------------------------------------- refusals of the C ABI (no GPU)

A, MIS = 0x10000, 0x10001   # addresses that are never read: the checks come before any CUDA call


def message(lib):
    return lib.lb_last_error().decode()


def test_no_warp_of_the_chunk_kernels_meets_others_on_the_way():
    """Every wait is bounded, and a warp whose wait gave up leaves its loop. A barrier among some of a CTA's warps inside such
    a loop would then hold the others for good, so these kernels have none: warps meet at the CTA's or the cluster's
    barriers, which each reaches whatever its waits returned. (Read from the source: no valid call makes a wait give up.)"""
    for name in ("lb_w8.cu", "lb_paged.cu"):
        source = (_lib.LIB_PATH.parent.parent / "csrc" / name).read_text()
        assert "named_barrier(" not in source and "bar.sync" not in source and "barrier.sync" not in source, name


def test_w8_abi_refusals():
    lib = _lib.load_library()
    q = lambda x=A, t=0, m=1, k=64, ldx=64, out=A, ldq=64, s=A: lib.lb_w8_quantize_rows(x, t, m, k, ldx, out, ldq, s, None)
    assert q(x=None) == 1 and "null" in message(lib)
    assert q(t=3) == 1 and q(m=0) == 1 and q(k=0) == 1 and q(ldx=63) == 1 and q(ldq=72) == 1 and q(ldq=48) == 1
    assert q(k=131073, ldx=131073, ldq=131088) == 1 and "131072" in message(lib)
    assert q(x=MIS) == 2 and q(out=MIS) == 2 and q(x=A + 2, t=2) == 2
    lin = lambda t=0, w=A, ldw=64, b=None, y=A, m=1, n=8, k=64, ws=A, wsb=1 << 30: lib.lb_w8_linear(
        A, t, k, w, ldw, A, b, y, m, n, k, ws, wsb, None)
    assert lin(t=2) == 1 and lin(w=None) == 1 and lin(n=0) == 1 and lin(w=MIS) == 2 and lin(b=MIS) == 2 and lin(y=MIS) == 2
    assert lib.lb_w8_workspace(0, 8, 64) == 0
    need = lib.lb_w8_workspace(300, 8, 64)
    assert need > 0 and lin(m=300, wsb=need - 1) == 1 and "workspace" in message(lib)
    assert lin(m=300, ws=MIS) == 2


def test_paged_abi_refusals():
    lib = _lib.load_library()

    def cache(**kw):
        f = dict(k=A, v=A, k_page_stride=2 * 16 * 64, v_page_stride=2 * 16 * 64, num_pages=4, dtype=0, nkv=2, hd=64, page_size=16)
        f.update(kw)
        return ctypes.addressof(_keep(_lib.PagedCacheStruct(**f)))

    kept = []

    def _keep(s):
        kept.append(s)
        return s

    def append(c=None, ld=8 * 64, t=1, nh=4, qn=None, kn=None, f=A, rot=64, **kw):
        return lib.lb_paged_norm_rope_append(A, ld, t, nh, qn, kn, 1e-6, f, rot, A, A, c or cache(**kw), A, None)

    for kw in (dict(k=None), dict(dtype=2), dict(nkv=0), dict(num_pages=0), dict(page_size=24), dict(page_size=0), dict(hd=72),
               dict(hd=272), dict(k_page_stride=64), dict(v_page_stride=2 * 16 * 64 + 4), dict(num_pages=2 ** 31),
               dict(qn=A), dict(t=0), dict(nh=0), dict(rot=24), dict(rot=80), dict(rot=-16), dict(ld=500), dict(ld=8 * 64 + 4),
               dict(f=None)):
        assert append(**kw) == 1, kw
    assert append(k=A + 8) == 2

    def attend(q=A, ts=256, hs=64, t=4, nh=4, width=3, stride=3, seqs=2, max_new=1, max_len=9, out=A, ots=256, ws=A,
               wsb=1 << 40, **kw):
        return lib.lb_paged_attention(q, ts, hs, t, nh, cache(**kw), A, stride, width, A, A, seqs, max_new, max_len, 0.1, out,
                                      ots, ws, wsb, None)

    for kw in (dict(q=None), dict(hd=32, k_page_stride=2 * 16 * 64), dict(nh=3), dict(nh=0), dict(t=0), dict(seqs=0), dict(width=0),
               dict(stride=2), dict(max_new=0), dict(max_len=0), dict(ts=100), dict(hs=60), dict(ots=128), dict(width=2 ** 30, stride=2 ** 30)):
        assert attend(**kw) == 1, kw
    assert attend(q=A + 8) == 2 and attend(out=MIS) == 2 and attend(ws=A + 8) == 2
    long = dict(seqs=1, width=4096, stride=4096, max_len=65536)
    assert attend(wsb=0, **long) == 1 and "workspace" in message(lib)
