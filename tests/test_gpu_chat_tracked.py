"""Tracked weights where the model's steps are fused, captured, or sharded by KV head."""

import pytest
import torch

from gpu_util import rel_l2
from test_gpu_chat import SYS, VIS, build, embeds, four_bits, positions, prompt      # noqa: F401 (four_bits: a fixture)

pytestmark = pytest.mark.gpu


def test_fused_decoder_in_a_graph():
    """The captured decoder as it is by default, with fused steps, against the same steps one by one.  The first layer sees the same
    queries and keys on both sides: its weights differ by fp32 roundings.  The second one's may be rounded the other way on their way there: queries and
    keys off by half a bfloat16 step, 2^-9, each, scores below 2 by 2 * 2 * 2^-9, and e to that and to the log-sum-exp's as much is 1 + 2^-6."""
    from calibquant_b200 import internlm2, patch_internvl as pi
    results = []
    for graphed in (False, True):
        shell = build(layers=2)
        pi.track_key_weights(shell)
        lm = shell.language_model
        (logits, past), at = prompt(shell, text=17)
        _, past = lm.forward_step(embeds(2, 4, shell, 3), positions(2, at, 4), past)
        tok = logits[:, -1].argmax(-1)
        if graphed:
            dec = internlm2.GraphedDecoder(lm, past, tok, at + 4, 12)
            assert dec.fused
            tokens = torch.cat([tok[:, None], dec.run(6)], 1)
            dec.close()
        else:
            tokens = [tok]
            for i in range(6):
                tok = lm.decode_token_fused(lm.model.tok_embeddings(tok).unsqueeze(1), positions(2, at + 4 + i, 1), past)
                past = [layer.attention._text_cache.views() for layer in lm.model.layers]
                tokens.append(tok)
            tokens = torch.stack(tokens, 1)
        n = SYS + 17 + 4 + 6
        results.append((tokens, [(a._key_weights[0], a._key_weights[1][:, :, :n]) for a in (l.attention for l in lm.model.layers)]))
        assert all(a._text_cache.length == n for a in (l.attention for l in lm.model.layers))
        past = pi.evict_cache(shell, keep_groups=1, keep_tokens=SYS + 9, recent=5)      # and on after it
        out = lm.forward_step_fused(embeds(2, 1, shell, 9), positions(2, at + 10, 1), past)
        assert torch.isfinite(out.float()).all()
    (t0, w0), (t1, w1) = results
    assert torch.equal(t0, t1)
    for rtol, a, b in zip((1e-5, 2.0 ** -6), w0, w1):
        for x, y in zip(a, b):
            assert torch.allclose(x, y, rtol=rtol, atol=1e-6)


def test_kv_heads_of_two_ranks():
    """A layer cut in two by KV head (one rank after the other): each rank has the weights of its heads, which the whole layer has too, evicts by
    them, and the ranks' partial results add up to the whole layer's.  Roundings of the type on either side as for a mask: 8 * 2^-9."""
    from calibquant_b200 import patch_internvl as pi, tp
    kw = dict(layers=1, heads=8, kv=4)

    def conversation(shell):
        pi.track_key_weights(shell)
        attn = shell.language_model.model.layers[0].attention
        x, outs, at = embeds(2, SYS + VIS + 20, shell, 1), [], SYS + VIS + 20
        y, _, past = attn(x, position_ids=positions(2, 0, at), use_cache=True)
        outs.append(y)
        for n in (9, 1, 40):
            y, _, past = attn(embeds(2, n, shell, n), position_ids=positions(2, at, n), past_key_value=past, use_cache=True)
            outs.append(y)
            at += n
        weights = [t.clone() for t in attn._key_weights]
        past = pi.evict_cache(shell, keep_groups=2, keep_tokens=SYS + 30, recent=10)[0]
        for n in (7, 1):
            y, _, past = attn(embeds(2, n, shell, n), position_ids=positions(2, at, n), past_key_value=past, use_cache=True)
            outs.append(y)
            at += n
        return outs, weights, attn.k_pack, past

    whole = conversation(build(**kw))
    ranks = []
    for rank in range(2):
        shell = build(**kw)
        tp.shard_layer_(shell.language_model.model.layers[0], rank, 2)
        ranks.append(conversation(shell))
    for rank, (_, weights, k_pack, past) in enumerate(ranks):
        mine = slice(2 * rank, 2 * rank + 2)
        for got, want in zip(weights, whole[1]):
            assert torch.allclose(got, want[:, mine], rtol=1e-5, atol=1e-6)
        assert torch.equal(k_pack[0], whole[2][0][:, mine])
        assert torch.equal(past[0][:, :, :SYS + 30], whole[3][0][:, mine, :SYS + 30])
    for y, a, b in zip(whole[0], ranks[0][0], ranks[1][0]):
        assert rel_l2(a.float() + b.float(), y) <= 8 * 2.0 ** -9
