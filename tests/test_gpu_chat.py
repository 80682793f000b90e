"""A conversation on one cached picture through the patched model: prompt, single tokens, a second question at once, weights of the keys,
eviction, and on with what is left."""

import pytest
import torch

from gpu_util import rel_l2

pytestmark = pytest.mark.gpu
VIS, SYS = 128, 41


@pytest.fixture(autouse=True)
def four_bits(monkeypatch):
    from calibquant_b200 import patch_internvl as pi
    monkeypatch.setattr(pi, "BITS_KV", 4)
    monkeypatch.setattr(pi, "KV_FORMAT", "group")
    monkeypatch.setenv("IMAGE_TOKEN_NUM", str(VIS))


def build(dtype=torch.bfloat16, layers=2, heads=8, kv=2, vocab=320, seed=0):
    from calibquant_b200 import internlm2, patch_internvl
    cfg = internlm2.InternLM2Config(hidden_size=heads * 128, num_attention_heads=heads, num_key_value_heads=kv, intermediate_size=512,
                                    num_hidden_layers=layers, vocab_size=vocab)
    shell = internlm2.ChatModelShell(cfg)
    internlm2.init_weights_(shell, seed)
    shell = shell.to("cuda", dtype).eval()
    patch_internvl.patch_model(shell, "calibquant")
    return shell


def embeds(B, T, shell, seed):
    g = torch.Generator().manual_seed(seed)
    lm = shell.language_model
    return torch.randn(B, T, lm.config.hidden_size, generator=g).to("cuda", lm.output.weight.dtype)


def positions(B, start, n):
    return torch.arange(start, start + n, device="cuda").expand(B, n)


def prompt(shell, B=2, text=20, seed=1):
    lm = shell.language_model
    x = embeds(B, SYS + VIS + text, shell, seed)
    return lm.forward_step(x, positions(B, 0, x.shape[1]), None), x.shape[1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,heads,kv", [(2, 8, 2), (19, 8, 2), (70, 12, 2), (300, 4, 4)])
def test_a_second_question_equals_its_tokens_one_by_one(n, heads, kv, dtype):
    from calibquant_b200 import ops
    shell = build(dtype, heads=heads, kv=kv)
    lm = shell.language_model
    (logits, past), at = prompt(shell)
    x = embeds(2, n, shell, 7)
    together, past_t = lm.forward_step(x, positions(2, at, n), past)
    assert past_t[0][0].shape == (2, kv, SYS + 20 + n, 128)
    (logits, past), at = prompt(shell)
    for i in range(n):
        one, past = lm.forward_step(x[:, i:i + 1], positions(2, at + i, 1), past)
    assert rel_l2(together, one) < 2e-2
    assert rel_l2(past_t[1][0], past[1][0]) < 2e-2       # the second layer's keys, of all new tokens
    # and on from there with a single token
    y = embeds(2, 1, shell, 8)
    (_, past2), at = prompt(shell)
    _, past2 = lm.forward_step(x, positions(2, at, n), past2)
    a, _ = lm.forward_step(y, positions(2, at + n, 1), past2)
    assert torch.isfinite(a.float()).all() and ops.device_status() == 0


def test_padding_mask_of_a_chunk():
    """The mask's last row says which keys count; a key that nobody sees might as well not be there.  With and without a mask the
    probabilities are rounded from numbers that differ in fp32's last bits, so the two agree to roundings of the type, not to the bit: half a step
    (2^-9) each for probabilities, unpacked values, attention and projection on either side, 8 * 2^-9 in all."""
    shell = build()
    lm, attn = shell.language_model, shell.language_model.model.layers[0].attention
    (_, past), at = prompt(shell)
    x = embeds(2, 6, shell, 3)
    keys = at + 6
    mask = torch.zeros(2, 1, 6, keys, device="cuda", dtype=x.dtype)
    mask[:, :, :, at:] = torch.triu(torch.full((6, 6), -torch.inf, device="cuda"), 1)
    plain, _, _ = attn(x, attention_mask=mask, position_ids=positions(2, at, 6), past_key_value=past[0], use_cache=True)
    attn._text_cache.length -= 6
    none, _, _ = attn(x, position_ids=positions(2, at, 6), past_key_value=past[0], use_cache=True)
    assert rel_l2(plain, none) <= 8 * 2.0 ** -9
    attn._text_cache.length -= 6
    mask[0, :, :, SYS + VIS:SYS + VIS + 5] = -torch.inf
    attn._text_cache.v[0, :, SYS:SYS + 5] = torch.nan
    padded, _, _ = attn(x, attention_mask=mask, position_ids=positions(2, at, 6), past_key_value=past[0], use_cache=True)
    assert torch.isfinite(padded.float()).all() and rel_l2(padded[1], none[1]) <= 8 * 2.0 ** -9 and not torch.equal(padded[0], none[0])
    with pytest.raises(ValueError):
        attn(x, attention_mask=mask[..., :-1], position_ids=positions(2, at, 6), past_key_value=past[0])


def test_what_is_tracked():
    """Every query of the question, the tokens and the second question gives each of its heads' weights once: their sum is known."""
    from calibquant_b200 import patch_internvl as pi
    shell = build()
    pi.track_key_weights(shell)
    lm = shell.language_model
    (_, past), at = prompt(shell, text=20)
    for i in range(3):
        _, past = lm.forward_step(embeds(2, 1, shell, i), positions(2, at + i, 1), past)
    _, past = lm.forward_step(embeds(2, 300, shell, 9), positions(2, at + 3, 300), past)      # the cache grows on the way
    for layer in lm.model.layers:
        w_vis, w_fp = layer.attention._key_weights
        total = (w_vis.double().sum(-1) + w_fp.double().sum(-1)).cpu()
        assert torch.allclose(total, torch.full_like(total, 4 * (20 + 3 + 300)), rtol=1e-4)
        assert not w_fp[:, :, layer.attention._text_cache.length:].any()
    (_, past), at = prompt(shell, text=0)                                                     # a new prompt starts anew
    assert lm.model.layers[0].attention._key_weights is None


def test_eviction_and_on():
    """Everything kept: the same numbers as before.  Less: the attention over what was kept, by the module and by hand."""
    from calibquant_b200 import ops, patch_internvl as pi
    import chunk_reference as ref
    shell = build()
    pi.track_key_weights(shell)
    lm = shell.language_model
    x = embeds(2, 5, shell, 2)

    def until_eviction():
        (_, past), at = prompt(shell, text=30)
        _, past = lm.forward_step(embeds(2, 40, shell, 3), positions(2, at, 40), past)
        return past, at + 40
    past, at = until_eviction()
    want, _ = lm.forward_step(x, positions(2, at, 5), past)
    until_eviction()
    past = pi.evict_cache(shell, keep_groups=VIS // 32, keep_tokens=SYS + 70)
    got, _ = lm.forward_step(x, positions(2, at, 5), past)
    assert torch.equal(got, want)

    past, at = until_eviction()
    attn = lm.model.layers[0].attention
    before = (attn.k_pack, attn.v_pack, attn._text_cache.k.clone(), attn._text_cache.v.clone(), attn._text_cache.length, [t.clone() for t in attn._key_weights])
    past = pi.evict_cache(shell, keep_groups=2, keep_tokens=SYS + 30, recent=10)
    assert past[0][0].shape[2] == SYS + 30 and attn.k_pack[1].shape[3] == 2
    groups = ref.kept_largest(before[5][0].cpu().double().unflatten(-1, (-1, 32)).sum(-1), 2)
    rank = before[5][1][:, :, :before[4]].clone()
    rank[:, :, :SYS] = rank[:, :, before[4] - 10:] = torch.inf
    tokens = ref.kept_largest(rank.cpu(), SYS + 30)
    assert torch.equal(past[0][0].cpu(), before[2][:, :, :before[4]].cpu().gather(2, tokens[..., None].expand(-1, -1, -1, 128)))
    idx = (groups[..., None] * 32 + torch.arange(32)).flatten(2)
    assert torch.equal(attn.v_pack[0].cpu(), before[1][0].cpu().gather(2, idx[..., None].expand(-1, -1, -1, 16)))
    # positions go on; a mask has no place any more
    out, _ = lm.forward_step(x, positions(2, at, 5), past)
    assert torch.isfinite(out.float()).all() and attn._text_cache.length == SYS + 35
    one, _ = lm.forward_step(x[:, :1], positions(2, at + 5, 1), [l.attention._text_cache.views() for l in lm.model.layers])
    assert torch.isfinite(one.float()).all()
    with pytest.raises(ValueError):
        attn(x, attention_mask=torch.zeros(2, 1, 5, 9, device="cuda"), position_ids=positions(2, at, 5), past_key_value=past[0])
    assert ops.device_status() == 0


def test_tracked_decoder_in_a_graph():
    """The captured decoder appends, attends and adds up weights as the eager steps do.  The first layer sees the same queries and keys on both
    sides: its weights differ by fp32 roundings.  What it passes on may be rounded the other way where partial results were merged
    in another order, so that the next layer's queries and keys are each off by half a bfloat16 step, 2^-9 of their size, and
    its scores, which are below 2 with these weights, by 2 * 2 * 2^-9 at most: e to that, and to the log-sum-exp's as much, is 1 + 2^-6."""
    from calibquant_b200 import internlm2, patch_internvl as pi
    results = []
    for graphed in (False, True):
        shell = build(layers=2)
        pi.track_key_weights(shell)
        lm = shell.language_model
        (logits, past), at = prompt(shell, text=17)
        tok = logits[:, -1].argmax(-1)
        if graphed:
            dec = internlm2.GraphedDecoder(lm, past, tok, at, 12, fused=False)
            tokens = torch.cat([tok[:, None], dec.run(6)], 1)
            dec.close()
        else:
            tokens = [tok]
            for i in range(6):
                logits, past = lm.forward_step(lm.model.tok_embeddings(tok).unsqueeze(1), positions(2, at + i, 1), past)
                tok = logits[:, -1].argmax(-1)
                tokens.append(tok)
            tokens = torch.stack(tokens, 1)
        n = SYS + 17 + 6
        results.append((tokens, [(a._key_weights[0], a._key_weights[1][:, :, :n]) for a in (l.attention for l in lm.model.layers)]))
    (t0, w0), (t1, w1) = results
    assert torch.equal(t0, t1)
    for rtol, a, b in zip((1e-5, 2.0 ** -6), w0, w1):
        for x, y in zip(a, b):
            assert torch.allclose(x, y, rtol=rtol, atol=1e-6)


def test_what_is_not_served(monkeypatch):
    from calibquant_b200 import patch_internvl as pi
    monkeypatch.setattr(pi, "BITS_KV", 2)
    shell = build()
    lm = shell.language_model
    (_, past), at = prompt(shell)
    with pytest.raises(NotImplementedError):
        lm.forward_step(embeds(2, 3, shell, 1), positions(2, at, 3), past)
    with pytest.raises(ValueError):
        pi.evict_cache(shell, keep_groups=1)
    monkeypatch.setattr(pi, "KV_FORMAT", "uint8")
    (_, past), at = prompt(shell)
    with pytest.raises(NotImplementedError):
        lm.forward_step(embeds(2, 3, shell, 1), positions(2, at, 3), past)


def test_an_open_decoder_keeps_cache_and_weights():
    """What would move or drop what a captured graph writes is refused until the decoder is closed; a prompt in between is not."""
    from calibquant_b200 import internlm2, patch_internvl as pi
    shell = build()
    pi.track_key_weights(shell)
    lm = shell.language_model
    (logits, past), at = prompt(shell, text=17)
    dec = internlm2.GraphedDecoder(lm, past, logits[:, -1].argmax(-1), at, 12, fused=False)
    attn = lm.model.layers[0].attention
    weights, before = attn._key_weights, [t.clone() for t in attn._key_weights]
    for refused in (lambda: lm.forward_step(embeds(2, 3, shell, 1), positions(2, at, 3), past), lambda: pi.track_key_weights(shell, False),
                    lambda: pi.track_key_weights(shell), lambda: pi.evict_cache(shell, keep_groups=1)):
        with pytest.raises(ValueError):
            refused()
    assert attn._key_weights is weights and all(torch.equal(a, b) for a, b in zip(weights, before))
    dec.run(2)
    assert not torch.equal(weights[1], before[1])
    ids = [t.data_ptr() for t in weights]
    del weights
    prompt(shell, text=5)                          # its layers start new caches and weights, those of the graph stay
    assert [t.data_ptr() for t in dec.held[0][3]] == ids
    dec.run(1)
    torch.cuda.synchronize()


def test_a_refused_eviction_changes_nothing():
    from calibquant_b200 import patch_internvl as pi
    shell = build(layers=2)
    pi.track_key_weights(shell)
    (_, past), _ = prompt(shell, text=20)
    layers = [l.attention for l in shell.language_model.model.layers]
    before = [(a.k_pack, a.v_pack, a._text_cache, a._text_cache.length, a._key_weights) for a in layers]
    n = SYS + 20
    for kw in (dict(keep_groups=0), dict(keep_groups=VIS // 32 + 1), dict(keep_groups=1, keep_tokens=n + 1), dict(keep_groups=1, keep_tokens=SYS + 3, recent=4),
               dict(keep_groups=1, keep_tokens=0, recent=0), dict(keep_groups=1, keep_tokens=n, recent=-1)):
        with pytest.raises(ValueError):
            pi.evict_cache(shell, **kw)
    for a, b in zip(layers, before):
        assert all(x is y for x, y in zip((a.k_pack, a.v_pack, a._text_cache, a._text_cache.length, a._key_weights), b)) and a._evicted == 0
    pi.evict_cache(shell, keep_groups=1, keep_tokens=SYS + 4, recent=4)
    assert all(a._text_cache.length == SYS + 4 for a in layers)
