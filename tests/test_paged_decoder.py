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
