"""PagedDecoder: the chunk operators together in a small decoder, against a plain float64 decoder over the same weights
(dequantized), and its page bookkeeping. INT4 weights leave only rounding between the two. With 8-bit integers the plain
decoder quantizes the activations as the operator is defined, and rounds to the type where the decoder stores: a value
that one rounding moves past the middle of a step is a whole step away, so the two have to round alike."""
import copy

import pytest
import torch

TINY = dict(hidden_size=256, intermediate_size=640, num_hidden_layers=2, num_attention_heads=4,
            num_key_value_heads=2, vocab_size=1024, tie_word_embeddings=True)


class Norm(torch.nn.Module):
    def __init__(self, n, seed):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        self.weight = torch.nn.Parameter((1 + 0.2 * torch.randn(n, generator=g)).half().cuda())


def tiny(norms=False, dtype=torch.float16, seed=4):
    from lowbit import decode
    m = decode.build(TINY, seed=seed).to(dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for i, layer in enumerate(m.model.layers):
        for p in (layer.self_attn.q_proj, layer.self_attn.k_proj, layer.self_attn.v_proj):
            p.bias.data.copy_(torch.randn(p.bias.shape, device="cuda", generator=g) * 0.1)
        for lin in (layer.self_attn.q_proj, layer.self_attn.k_proj):
            lin.weight.data *= 6   # scores that are not all alike
        if norms:
            layer.self_attn.q_norm, layer.self_attn.k_norm = Norm(64, 10 + i).to(dtype), Norm(64, 20 + i).to(dtype)
    return m


@torch.no_grad()
def plain_logits(model, ids, weights):
    """Logits after every token in float64, projections dequantized from the decoder's own format."""
    from lowbit import ops
    cfg, nh, nkv, hd = model.config, 4, 2, 64
    dtype = model.lm_head.weight.dtype

    def stored(v):
        return v.to(dtype).double() if weights == "w8" else v

    def weight(lin):
        if weights == "w4":
            return ops.dequantize_w4_gpu(*ops.quantize_w4_gpu(lin.weight)).double()
        q, s = ops.quantize_w8_gpu(lin.weight)
        return q.double() * s.double()[:, None]

    def product(x, lin):
        if weights == "w8":   # activations too, as the operator is defined
            amax = x.abs().amax(-1, keepdim=True)
            x = torch.round(x * 127 / amax) * (amax / 127)
        y = x @ weight(lin).t()
        return stored(y if lin.bias is None else y + lin.bias.double())

    def rms(x, w):
        return stored(stored(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps)) * w.double())

    t = len(ids)
    x = model.model.embed_tokens.weight[ids].double()
    freq = 1.0 / 1e6 ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    angle = torch.arange(t, device="cuda", dtype=torch.float64)[:, None, None] * freq
    mask = torch.ones(t, t, device="cuda", dtype=torch.bool).triu(1)

    def rope(h):
        a, b = h.chunk(2, -1)
        return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)

    for layer in model.model.layers:
        a, m = layer.self_attn, layer.mlp
        h = rms(x, layer.input_layernorm.weight)
        q, k, v = (product(h, p).view(t, -1, hd) for p in (a.q_proj, a.k_proj, a.v_proj))
        if hasattr(a, "q_norm"):
            q, k = (h * torch.rsqrt(h.square().mean(-1, keepdim=True) + cfg.rms_norm_eps) * n.weight.double()
                    for h, n in ((q, a.q_norm), (k, a.k_norm)))
        q, k = stored(rope(q)), stored(rope(k))
        k, v = k.repeat_interleave(nh // nkv, 1), v.repeat_interleave(nh // nkv, 1)
        s = torch.einsum("qhd,khd->hqk", q, k) / 8
        p = torch.softmax(s.masked_fill(mask, float("-inf")), -1)
        x = stored(x + product(stored(torch.einsum("hqk,khd->qhd", p, v).reshape(t, nh * hd)), a.o_proj))
        h = rms(x, layer.post_attention_layernorm.weight)
        act = stored(stored(torch.nn.functional.silu(product(h, m.gate_proj))) * product(h, m.up_proj))
        x = stored(x + product(act, m.down_proj))
    return rms(x, model.model.norm.weight) @ model.lm_head.weight.double().t()


def feed(dec, ids, pieces):
    """The logits after each piece of ids, fed in turn."""
    sid, rows, at = dec.open(), [], 0
    for n in pieces:
        rows.append(dec.forward({sid: ids[at:at + n]})[0])
        at += n
    dec.close(sid)
    return torch.stack(rows)


@pytest.mark.gpu
@pytest.mark.parametrize("weights,norms,dtype,bar", [("w4", False, torch.float16, 2e-2), ("w4", True, torch.float16, 2e-2),
                                                     ("w8", True, torch.float16, 8e-2), ("w8", False, torch.bfloat16, 1.2e-1)])
def test_paged_decoder_matches_a_plain_decoder(weights, norms, dtype, bar):
    from lowbit import ops, paged
    model = tiny(norms, dtype)
    dec = paged.PagedDecoder(model, num_pages=32, page_size=16, weights=weights)
    ids = torch.randint(0, 1024, (150,), generator=torch.Generator().manual_seed(9)).tolist()
    want = plain_logits(model, ids, weights)
    rms = want.square().mean().sqrt()
    for pieces in ([150], [1] * 20 + [130], [100, 1, 49], [17, 64, 1, 68]):
        got = feed(dec, ids, pieces)
        ends = torch.tensor(pieces).cumsum(0) - 1
        err = ((got.double() - want[ends]).abs().max() / rms).item()
        assert err < bar, (pieces, err)
    assert len(dec._free) == 32 and ops.ext().lib.lb_device_error() == 0


@pytest.mark.gpu
def test_sequences_of_a_batch_do_not_touch_each_other():
    """Several sequences in one call, chunks and single tokens mixed, give what each gives alone; pages come back."""
    from lowbit import paged
    dec = paged.PagedDecoder(tiny(), num_pages=24, page_size=16, weights="w4")
    g = torch.Generator().manual_seed(2)
    texts = [torch.randint(0, 1024, (n,), generator=g).tolist() for n in (40, 7, 90)]
    alone = [feed(dec, ids, [len(ids) - 1, 1])[-1] for ids in texts]
    sids = [dec.open() for _ in texts]
    dec.forward({s: ids[:-1] for s, ids in zip(sids, texts)})
    dec.close(sids.pop(1))
    again = dec.open()
    out = dec.forward({sids[0]: texts[0][-1:], again: texts[1], sids[1]: texts[2][-1:]})
    scale = torch.stack(alone).float().square().mean().sqrt()
    for row, want in zip(out, (alone[0], alone[1], alone[2])):
        assert ((row.float() - want.float()).abs().max() / scale).item() < 2e-2
    with pytest.raises(RuntimeError, match="pages"):
        dec.forward({sids[0]: list(range(400))})
    with pytest.raises(ValueError):
        dec.forward({})
    with pytest.raises(ValueError):
        paged.PagedDecoder(tiny(dtype=torch.bfloat16), 4, weights="w4")


# ------------------------------------------------------------------------------- what the decoders refuse (no GPU)

def empty_model(**kw):
    """A model as far as the refusals look: its config, and attention modules without weights."""
    from types import SimpleNamespace as Ns
    from lowbit import decode
    return Ns(config=decode.qwen2_config(TINY, **kw), model=Ns(layers=[Ns(self_attn=Ns()) for _ in range(2)]))


REFUSED = [dict(rope_parameters={"rope_type": "linear", "factor": 4.0, "rope_theta": 1e6}),
           dict(rope_parameters={"rope_type": "yarn", "factor": 4.0, "rope_theta": 1e6, "original_max_position_embeddings": 8192}),
           dict(rope_parameters={"rope_type": "llama3", "factor": 8.0, "rope_theta": 5e5, "low_freq_factor": 1.0,
                                 "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}),
           dict(hidden_act="gelu")]


@pytest.mark.parametrize("kw", REFUSED)
def test_decoders_refuse_models_that_they_would_compute_wrongly(kw):
    from lowbit import decode, paged
    with pytest.raises(ValueError, match="not supported"):
        paged.PagedDecoder(empty_model(**kw), num_pages=4)
    with pytest.raises(ValueError, match="not supported"):
        decode.Int4Decoder(empty_model(**kw), 64)


def test_int4_decoder_refuses_head_dims_and_norms_that_it_ignores():
    from types import SimpleNamespace as Ns
    from lowbit import decode
    with pytest.raises(ValueError, match="head_dim"):
        decode.Int4Decoder(empty_model(head_dim=128), 64)
    normed = empty_model()
    normed.model.layers[1].self_attn = Ns(q_norm=None)
    with pytest.raises(ValueError, match="norms"):
        decode.Int4Decoder(normed, 64)


def test_paged_decoder_refuses_head_dims_of_the_attention():
    from lowbit import paged
    model = empty_model(head_dim=32)
    model.model.embed_tokens = torch.nn.Embedding(4, 4)
    with pytest.raises(ValueError, match="64 and 128"):
        paged.PagedDecoder(model, num_pages=4)


WINDOW = dict(use_sliding_window=True, sliding_window=64, max_window_layers=1)
DYNAMIC = dict(rope_parameters={"rope_type": "dynamic", "factor": 4.0, "rope_theta": 1e6}, max_position_embeddings=64)


@pytest.mark.parametrize("kw", [WINDOW, DYNAMIC])
def test_decoders_stop_where_a_window_or_scaled_angles_begin(kw):
    from lowbit import decode, paged
    assert decode.context_limit(empty_model(**kw).config) == 64
    assert decode.context_limit(empty_model(use_sliding_window=False, sliding_window=64).config) is None
    with pytest.raises(ValueError, match="64 tokens"):
        decode.Int4Decoder(empty_model(**kw), 65)
    dec = bookkeeper(limit=64)
    sid = dec.open()
    for n in (60, 4):
        dec.forward({sid: [1] * n})
    with pytest.raises(ValueError, match="65 tokens"):
        dec.forward({sid: [1]})


def bookkeeper(limit=None, pages=10):
    """A PagedDecoder without layers, on the CPU: its page bookkeeping, its embedding and its head."""
    from lowbit import paged
    dec = paged.PagedDecoder.__new__(paged.PagedDecoder)
    dec.page_size, dec.limit, dec.device, dec.dtype, dec.layers, dec.eps = 16, limit, torch.device("cpu"), torch.float32, [], 1e-6
    dec.embed, dec.head, dec.norm = torch.randn(32, 8), torch.randn(32, 8), torch.ones(8)
    dec._free, dec._seqs, dec._next = list(range(pages - 1, -1, -1)), {}, 0
    return dec


def test_a_call_that_raises_changes_no_sequence():
    dec = bookkeeper()
    a, b = dec.open(), dec.open()
    dec.forward({a: [1] * 20, b: [2]})
    before = copy.deepcopy((dec._free, dec._seqs))
    with pytest.raises(ValueError):   # a token that is none, after a sequence in order
        dec.forward({a: [1] * 40, b: [4, "x"]})
    assert (dec._free, dec._seqs) == before
    norm, dec.norm = dec.norm, torch.ones(5)
    with pytest.raises(RuntimeError):   # the last of the call's products fails
        dec.forward({a: [1] * 40, b: [4]})
    assert (dec._free, dec._seqs) == before
    dec.norm = norm
    dec.forward({a: [1] * 40, b: [4] * 30})
    assert dec._seqs == {a: {"length": 60, "pages": [0, 1, 3, 4]}, b: {"length": 31, "pages": [2, 5]}}
    assert dec._free == [9, 8, 7, 6]
    dec.close(a)
    assert sorted(dec._free) == [0, 1, 3, 4, 6, 7, 8, 9]


@pytest.mark.parametrize("tok", [-1, 32, 2 ** 40, torch.tensor(32)])
def test_token_ids_outside_the_embedding_are_refused_before_any_work(tok):
    """On the host: -1 would read the last row, 32 of 32 fail in the lookup on the device."""
    dec = bookkeeper()
    a, b = dec.open(), dec.open()
    dec.forward({a: [0, 31]})
    before = copy.deepcopy((dec._free, dec._seqs))
    with pytest.raises(ValueError, match="token id"):
        dec.forward({b: [3], a: [1, tok]})
    assert (dec._free, dec._seqs) == before


@pytest.mark.gpu
def test_a_call_that_failed_in_a_layer_can_be_repeated(monkeypatch):
    from lowbit import paged
    dec = paged.PagedDecoder(tiny(), num_pages=16, page_size=16, weights="w8")
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 1024, (80,), generator=g).tolist()
    want = feed(dec, ids, [50, 30])
    sid = dec.open()
    first = dec.forward({sid: ids[:50]})
    state = copy.deepcopy((dec._free, dec._seqs))
    calls, attention = [], paged.attention

    def failing(*args, **kw):
        calls.append(1)
        if len(calls) == 2:
            raise torch.OutOfMemoryError("no memory")
        return attention(*args, **kw)

    monkeypatch.setattr(paged, "attention", failing)
    with pytest.raises(torch.OutOfMemoryError):
        dec.forward({sid: ids[50:]})
    assert (dec._free, dec._seqs) == state
    monkeypatch.undo()
    assert torch.equal(torch.cat((first, dec.forward({sid: ids[50:]}))), want)


# ------------------------------------------------------------------------------------- drafted trees, 8-bit floating point

@torch.no_grad()
def plain_f8_logits(model, ids, activations=True):
    """plain_logits with the projections of linear_f8: weights and (or not) activations quantized by blocks, as the operator is
    defined, values rounded to the model's type where the decoder stores them."""
    from lowbit import ops

    class Blocks(torch.nn.Module):
        def __init__(self, lin):
            super().__init__()
            q, s = ops.quantize_f8_gpu(lin.weight)
            n, k = q.shape
            self.w = q.double() * s.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
            self.bias = lin.bias

    dtype = model.lm_head.weight.dtype

    def product(x, b):
        if not activations:
            y = x @ b.w.t()
            return (y if b.bias is None else y + b.bias.double()).to(dtype).double()
        t, k = x.shape
        g = torch.nn.functional.pad(x, (0, -k % 128)).view(t, -1, 128)
        a = g.abs().amax(2, keepdim=True).clamp(min=2.0 ** -100)
        g = (g.float() * (448.0 / a).float()).to(torch.float8_e4m3fn).double() * (a / 448)
        y = g.reshape(t, -1)[:, :k] @ b.w.t()
        return (y if b.bias is None else y + b.bias.double()).to(dtype).double()

    def rms(x, w):
        return (((x * torch.rsqrt(x.square().mean(-1, keepdim=True) + model.config.rms_norm_eps)).to(dtype).double()) * w.double()).to(dtype).double()

    t, hd = len(ids), 64
    x = model.model.embed_tokens.weight[ids].double()
    freq = 1.0 / 1e6 ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    angle = torch.arange(t, device="cuda", dtype=torch.float64)[:, None, None] * freq
    mask = torch.ones(t, t, device="cuda", dtype=torch.bool).triu(1)
    for layer in model.model.layers:
        a, m = layer.self_attn, layer.mlp
        # the decoder quantizes q, k, v and gate, up as one weight each: blocks of 128 rows do not cross them at these sizes
        h = rms(x, layer.input_layernorm.weight)
        q, k, v = (product(h, Blocks(p)).view(t, -1, hd) for p in (a.q_proj, a.k_proj, a.v_proj))

        def rope(z):
            c, d = z.chunk(2, -1)
            return torch.cat((c * angle.cos() - d * angle.sin(), d * angle.cos() + c * angle.sin()), -1).to(dtype).double()

        q, k = rope(q), rope(k)
        k, v = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
        p = torch.softmax((torch.einsum("qhd,khd->hqk", q, k) / 8).masked_fill(mask, float("-inf")), -1)
        x = (x + product(torch.einsum("hqk,khd->qhd", p, v).reshape(t, -1).to(dtype).double(), Blocks(a.o_proj))).to(dtype).double()
        h = rms(x, layer.post_attention_layernorm.weight)
        act = (torch.nn.functional.silu(product(h, Blocks(m.gate_proj))).to(dtype).double() * product(h, Blocks(m.up_proj))).to(dtype).double()
        x = (x + product(act, Blocks(m.down_proj))).to(dtype).double()
    return rms(x, model.model.norm.weight) @ model.lm_head.weight.double().t()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_paged_decoder_with_f8_weights_is_as_near_as_a_plain_one(dtype):
    """An e4m3 step is up to 2^-3 of a value, and where a rounding of the stored type moves a value past the middle of a step, the
    decoder and a plain one go a whole step apart there: after a layer the two are as good as quantized independently. So neither is the
    other's measure; both have the same distance (root mean square, over more than 10^5 logits) from a decoder with the same
    weights whose activations are not quantized, to a quarter for what the stored type's own roundings add."""
    from lowbit import ops, paged
    model = tiny(dtype=dtype)
    dec = paged.PagedDecoder(model, num_pages=32, page_size=16, weights="f8")
    ids = torch.randint(0, 1024, (150,), generator=torch.Generator().manual_seed(9)).tolist()
    exact = plain_f8_logits(model, ids, activations=False)
    plain = (plain_f8_logits(model, ids) - exact).square().mean().sqrt().item()
    for pieces in ([1] * 150, [2] * 75):
        got = feed(dec, ids, pieces)
        ends = torch.tensor(pieces).cumsum(0) - 1
        mine = (got.double() - exact[ends]).square().mean().sqrt().item()
        assert mine < 1.25 * plain, (pieces[:2], mine, plain)
    whole = feed(dec, ids, [150])
    assert (whole.double() - exact[-1:]).square().mean().sqrt().item() < 2 * plain   # (1024 values of one row, not alike)
    assert len(dec._free) == 32 and ops.ext().lib.lb_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("weights", ["w4", "w8", "f8"])
def test_verify_keeps_what_the_model_would_have_chosen(weights):
    """Trees of right and wrong drafts, several sequences at once: every accepted token is, within the products' roundings, the largest
    logit of a decoder that is fed the same text plainly; a tree's cache then continues as that decoder's does. The bars are those of the
    tests against plain decoders; f8: an activation's error is 2^-3 / sqrt(12) / 1.44 = 2.5 % of it in the mean square (steps of 2^-4 to
    2^-3 of a value), so each product's, and six that add up in the residual stream give at most 6 %; two decoders are sqrt(2) times
    that apart, and of 10^4 values the largest at 4.5 times: 0.4."""
    from lowbit import ops, paged
    import random
    model = tiny()
    bar = {"w4": 2e-2, "w8": 8e-2, "f8": 4e-1}[weights]
    dec, ref = (paged.PagedDecoder(model, num_pages=64, page_size=16, weights=weights) for _ in range(2))
    rng = random.Random(5)
    sids = [dec.open() for _ in range(3)]
    texts = {s: [rng.randrange(1024) for _ in range(n)] for s, n in zip(sids, (5, 33, 16))}
    logits = dec.forward(dict(texts))
    nxt = {s: int(row.argmax()) for s, row in zip(sids, logits)}

    def greedy(text, n):   # what a plain decoder would say next, as drafts
        sid, out = ref.open(), []
        last = ref.forward({sid: text})[0]
        for _ in range(n):
            out.append(int(last.argmax()))
            last = ref.forward({sid: out[-1:]})[0]
        ref.close(sid)
        return out

    taken = 0
    for turn in range(4):
        trees = {}
        for s in sids:
            good = greedy(texts[s] + [nxt[s]], 3)
            # the right drafts among wrong ones, in levels: 1 2 3 after the first token, 4 5 after one of them, 6 after one of those
            first, second = rng.randint(1, 3), rng.randint(4, 5)
            tokens = [nxt[s]] + [rng.randrange(1024) for _ in range(6)]
            parents = [-1, 0, 0, 0, first, first, second]
            tokens[first], tokens[second], tokens[6] = good[0], good[1], good[2] if turn % 2 else (good[2] + 1) % 1024
            trees[s] = (tokens, parents)
        got = dec.verify(trees)
        for s in sids:
            new = [nxt[s]] + got[s][:-1]
            text = texts[s] + new
            assert dec._seqs[s]["length"] == len(text) and len(dec._seqs[s]["pages"]) == -(-len(text) // 16)
            sid = ref.open()
            rows = [ref.forward({sid: text[:len(texts[s]) + 1]})[0]] + [ref.forward({sid: [t]})[0] for t in new[1:]]
            ref.close(sid)
            for row, choice in zip(rows, got[s]):
                assert (row.max() - row[choice]).item() <= 2 * bar * row.float().square().mean().sqrt().item()
            texts[s], nxt[s] = text, got[s][-1]
            taken += len(got[s])
    assert taken > 2 * 3 * 4   # most of the right drafts were accepted
    # the caches hold the texts: their next logits are a plain decoder's
    out = dec.forward({s: [nxt[s]] for s in sids})
    for row, s in zip(out, sids):
        sid = ref.open()
        want = ref.forward({sid: texts[s] + [nxt[s]]})[0].float()
        ref.close(sid)
        assert ((row.float() - want).abs().max() / want.square().mean().sqrt()).item() < bar
    for s in sids:
        dec.close(s)
    assert sorted(dec._free) == list(range(64)) and ops.ext().lib.lb_device_error() == 0


@pytest.mark.parametrize("tree", [([], []), ([1], [-1, 0]), ([1, 2], [-1, 1]), ([1, 2], [-1, -1]), ([1, 2], [0, 0]), ([1, 2, 3], [-1, 2, 0]),
                                  ([32, 1], [-1, 0]), ([1, -1], [-1, 0]), ([1] * 1025, list(range(-1, 1024))), ([1] * 200, list(range(-1, 199)))])
def test_verify_refuses_what_is_no_tree_and_changes_nothing(tree):
    """Before any work: shapes, parents, token ids, and more tokens than pages."""
    dec = bookkeeper()
    a, b = dec.open(), dec.open()
    dec.forward({a: [1] * 20})
    before = copy.deepcopy((dec._free, dec._seqs))
    with pytest.raises((ValueError, RuntimeError)):
        dec.verify({b: ([3], [-1]), a: tree})
    with pytest.raises(ValueError):
        dec.verify({})
    assert (dec._free, dec._seqs) == before


def test_the_limit_of_a_model_holds_for_a_trees_levels_not_for_its_tokens(monkeypatch):
    """60 tokens of 64 and a tree of 30: with four levels the last token's context is 64, with five it is 65."""
    from lowbit import paged

    class Planned(Exception):
        pass

    def plan(*args, **kw):
        raise Planned

    monkeypatch.setattr(paged, "plan", plan)
    dec = bookkeeper(limit=64)
    sid, other = dec.open(), dec.open()
    dec.forward({sid: [1] * 60, other: [2] * 3})
    wide = [-1, 0, 1, 2] + [i % 3 for i in range(26)]
    before = copy.deepcopy((dec._free, dec._seqs))
    with pytest.raises(Planned):
        dec.verify({sid: ([1] * 30, wide), other: ([1] * 61, list(range(-1, 60)))})
    with pytest.raises(ValueError, match="65 tokens.*allows 64"):
        dec.verify({sid: ([1] * 30, wide[:-1] + [3])})
    with pytest.raises(ValueError, match="65 tokens.*allows 64"):
        dec.verify({sid: ([1], [-1]), other: ([1] * 62, list(range(-1, 61)))})
    assert (dec._free, dec._seqs) == before


def test_verification_moves_the_rows_of_however_many_layers(monkeypatch):
    """compact takes up to 128 caches a call."""
    from lowbit import paged
    dec, moved = bookkeeper(), []
    dec.layers = [{"cache": i} for i in range(300)]
    dec._layers = lambda x, *args: x
    vector = lambda *v: torch.tensor(v)
    monkeypatch.setattr(paged, "plan", lambda *args, **kw: paged.Plan(vector(0, 2), vector(2), vector(0, 1), vector(0, 1), None, None, None))
    monkeypatch.setattr(paged, "verify", lambda *args, **kw: paged.Verified(vector(2), vector(0, 1)[None], vector(7), vector(3, 7)))
    monkeypatch.setattr(paged, "compact", lambda caches, *args: (len(caches) <= 128 or pytest.fail("too many")) and moved.extend(caches))
    sid = dec.open()
    assert dec.verify({sid: ([1, 3], [-1, 0])}) == {sid: [3, 7]}
    assert moved == list(range(300)) and dec._seqs[sid]["length"] == 2


@pytest.mark.gpu
def test_a_wide_tree_at_the_models_limit_gives_what_it_gives_below_it():
    from lowbit import paged
    model = tiny()
    near, far = (paged.PagedDecoder(model, num_pages=16, page_size=16) for _ in range(2))
    near.limit, text, got = 40, [int(i) for i in torch.randint(0, 1024, (36,), generator=torch.Generator().manual_seed(2))], []
    for dec in (near, far):
        sid = dec.open()
        first = int(dec.forward({sid: text})[0].argmax())
        got.append(dec.verify({sid: ([first] + list(range(20)), [-1, 0, 1, 2] + [i % 3 for i in range(17)])})[sid])
        got[-1] += dec.forward({sid: got[-1][-1:]})[0].tolist() if dec._seqs[sid]["length"] < 40 else []
    assert got[0] == got[1]


@pytest.mark.gpu
def test_a_verification_that_failed_in_a_layer_can_be_repeated(monkeypatch):
    from lowbit import paged
    dec = paged.PagedDecoder(tiny(), num_pages=16, page_size=16, weights="f8")
    sid = dec.open()
    logits = dec.forward({sid: list(range(30))})
    tree = ([int(logits[0].argmax()), 5, 6, 7], [-1, 0, 1, 0])
    state = copy.deepcopy((dec._free, dec._seqs))
    calls, attention = [], paged.tree_attention

    def failing(*args, **kw):
        calls.append(1)
        if len(calls) == 2:
            raise torch.OutOfMemoryError("no memory")
        return attention(*args, **kw)

    monkeypatch.setattr(paged, "tree_attention", failing)
    with pytest.raises(torch.OutOfMemoryError):
        dec.verify({sid: tree})
    assert (dec._free, dec._seqs) == state
    monkeypatch.undo()
    other = paged.PagedDecoder(tiny(), num_pages=16, page_size=16, weights="f8")
    oid = other.open()
    other.forward({oid: list(range(30))})
    assert dec.verify({sid: tree})[sid] == other.verify({oid: tree})[oid]
