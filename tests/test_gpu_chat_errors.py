"""What the patched model refuses in a conversation, or fails at, leaves its caches and weights as they were."""

import pytest
import torch

from test_gpu_chat import SYS, VIS, build, embeds, four_bits, positions, prompt      # noqa: F401 (four_bits: a fixture)

pytestmark = pytest.mark.gpu


def attentions(shell):
    return [layer.attention for layer in shell.language_model.model.layers]


def state(shell):
    return [(a.k_pack, a.v_pack, a._text_cache, a._text_cache.length, a._key_weights, a._evicted, a._keys_differ) for a in attentions(shell)]


def same(a, b):
    return all(x is y or isinstance(x, (int, bool)) and x == y for s, t in zip(a, b) for x, y in zip(s, t))


def test_an_eviction_beyond_the_kernels_sizes():
    """More full-precision tokens than can be ranked: the groups of no layer are dropped either, and the conversation goes on."""
    from calibquant_b200 import patch_internvl as pi
    shell = build()
    pi.track_key_weights(shell)
    lm, n = shell.language_model, 24577 - SYS
    (_, past), at = prompt(shell, B=1, text=n)
    before = state(shell)
    with pytest.raises((ValueError, RuntimeError)):
        pi.evict_cache(shell, keep_groups=1, keep_tokens=SYS + 100)
    assert same(state(shell), before)
    _, past = lm.forward_step(embeds(1, 3, shell, 5), positions(1, at, 3), past)
    past = pi.evict_cache(shell, keep_groups=1)
    assert past[1][0].shape[2] == SYS + n + 3 and all(a.k_pack[1].shape[3] == 1 for a in attentions(shell))


@pytest.mark.parametrize("tracked", [False, True])
def test_a_chunk_that_is_refused_appends_nothing(tracked):
    from calibquant_b200 import patch_internvl as pi
    shell = build()
    pi.track_key_weights(shell, tracked)
    (_, past), at = prompt(shell)
    before, attn = state(shell), attentions(shell)[0]
    x = embeds(2, 5, shell, 1)
    with pytest.raises((RuntimeError, ValueError)):      # a mask that is not on the GPU
        attn(x, attention_mask=torch.zeros(2, 1, 5, at + 5), position_ids=positions(2, at, 5), past_key_value=past[0])
    assert same(state(shell), before)
    want, _, views = attn(x, position_ids=positions(2, at, 5), past_key_value=past[0], use_cache=True)
    assert views[0].shape[2] == SYS + 25 and torch.isfinite(want.float()).all()


@pytest.mark.parametrize("fmt,bits", [("group", 1), ("group", 2), ("uint8", 4), ("uint8", 2)])
def test_tracking_at_other_widths_changes_nothing(fmt, bits, monkeypatch):
    """Prompt, single tokens, several at once and the captured decoder are refused before a cache is replaced or appended to; without tracking they go on."""
    from calibquant_b200 import internlm2, patch_internvl as pi
    shell = build()
    lm = shell.language_model
    (_, past), at = prompt(shell)                     # 4 bits
    before = state(shell)
    monkeypatch.setattr(pi, "KV_FORMAT", fmt)
    monkeypatch.setattr(pi, "BITS_KV", bits)
    pi.track_key_weights(shell)
    with pytest.raises(NotImplementedError):
        prompt(shell)
    assert same(state(shell), before)
    pi.track_key_weights(shell, False)
    (logits, past), at = prompt(shell)
    one, tok = embeds(2, 1, shell, 1), logits[:, -1].argmax(-1)
    before, u8 = state(shell), [a._u8_state for a in attentions(shell)]
    pi.track_key_weights(shell)
    for call in (lambda: lm.forward_step(one, positions(2, at, 1), past), lambda: internlm2.GraphedDecoder(lm, past, tok, at, 8)):
        with pytest.raises(NotImplementedError):
            call()
        assert same(state(shell), before) and all(a._u8_state is u for a, u in zip(attentions(shell), u8))
    pi.track_key_weights(shell, False)
    with pytest.raises(NotImplementedError):
        lm.forward_step(embeds(2, 3, shell, 1), positions(2, at, 3), past)
    out, past = lm.forward_step(one, positions(2, at, 1), past)
    assert past[0][0].shape[2] == SYS + 21 and torch.isfinite(out.float()).all()


def test_masks_after_an_eviction():
    """Masks over keys go on as long as all keys are there, in their order; once some are dropped they are refused, whatever is kept later."""
    from calibquant_b200 import patch_internvl as pi
    shell = build()
    pi.track_key_weights(shell)
    (_, past), at = prompt(shell)
    attn = attentions(shell)[0]
    x, mask = embeds(2, 5, shell, 1), torch.zeros(2, 1, 5, at + 5, device="cuda")
    past = pi.evict_cache(shell, keep_groups=VIS // 32, keep_tokens=SYS + 20, recent=9)      # all of them
    out, _, views = attn(x, attention_mask=mask, position_ids=positions(2, at, 5), past_key_value=past[0], use_cache=True)
    assert torch.isfinite(out.float()).all() and views[0].shape[2] == SYS + 25
    one = torch.zeros(2, 1, 1, at + 6, device="cuda")
    _, _, views = attn(x[:, :1], attention_mask=one, position_ids=positions(2, at + 5, 1), past_key_value=views, use_cache=True)
    (_, past), at = prompt(shell)
    for kw in (dict(keep_tokens=SYS + 19, recent=9), dict(keep_groups=VIS // 32), dict(keep_tokens=SYS + 19, recent=9)):
        past = pi.evict_cache(shell, **kw)
        with pytest.raises(ValueError):
            attn(x, attention_mask=mask, position_ids=positions(2, at, 5), past_key_value=past[0])
        with pytest.raises(ValueError):
            attn(x[:, :1], attention_mask=one[..., :at + 1], position_ids=positions(2, at, 1), past_key_value=past[0])
    assert attn._text_cache.length == SYS + 19
