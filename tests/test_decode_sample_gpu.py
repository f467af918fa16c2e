"""Sampled generation on the runner (mlm_llama_decode_sample and its batch form): every
token equals the plain 64-bit sampling of the runner's own logits at that step."""
from __future__ import annotations

import numpy as np
import pytest

from metallm_b200 import Context, Llama, MLMError
from metallm_b200.synthetic import fill_llama, llama_config
from tests import kv4_reference as R

pytestmark = pytest.mark.gpu

SEED = 77
SETTINGS = [(0.8, 40, 0.95, 0.02), (1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 0, 0.9, 0.0)]


def _cfg(**kw):
    f = dict(n_layers=2, dim=1024, n_heads=8, n_kv_heads=2, ffn_dim=1024, vocab=5120, max_seq=64)
    f.update(kw)
    return llama_config(**f)


def _by_hand(ctx, m, token, settings, us):
    """The tokens that mlm_llama_forward's logits and the plain sampling give."""
    lg = ctx.alloc(4 * m.cfg.vocab)
    toks = []
    for u in us:
        m.forward(token, lg)
        token = R.sample(lg.download(np.float32), *settings, u)[0]
        toks.append(token)
    return toks


def test_decode_sample_matches_sampling_the_logits(ctx):
    m = Llama(ctx, _cfg())
    fill_llama(m, SEED)
    steps = 12
    out = ctx.alloc(4 * steps)
    for i, settings in enumerate(SETTINGS + SETTINGS[:1]):  # one captured step, many settings
        us = np.random.default_rng(i).random(steps).astype(np.float32)
        m.reset()
        want = _by_hand(ctx, m, 5 + i, settings, us)
        m.reset()
        m.decode_sample(5 + i, steps, settings, ctx.to_device(us), out)
        assert out.download(np.int32).tolist() == want, settings
        assert m.position == steps
        m.decode_sample(want[-1], 3, settings, ctx.to_device(us[:3]), out)  # goes on from there
        assert m.position == steps + 3
    m.close()


def test_greedy_and_sampled_steps_take_turns(ctx):
    """Temperature 0 is the greedy loop; both captured steps live side by side."""
    m = Llama(ctx, _cfg())
    fill_llama(m, SEED)
    a, b = ctx.alloc(4 * 8), ctx.alloc(4 * 8)
    u = ctx.to_device(np.full(8, 0.5, np.float32))
    for _ in range(2):
        m.reset()
        m.decode_greedy(3, 8, a)
        m.reset()
        m.decode_sample(3, 8, (0.0, 0, 1.0, 0.0), u, b)
        assert np.array_equal(a.download(np.int32), b.download(np.int32))
    m.close()


def test_decode_sample_batch(ctx):
    """Each sequence by its own settings and numbers: the batched step's logits sampled by
    hand.  One 256-weight block per row: the batched linears add one partial sum to each
    output, so that both runs' logits agree to the last bit."""
    B, steps = 4, 7
    m = Llama(ctx, _cfg(dim=256, n_heads=2, n_kv_heads=1, ffn_dim=256), batch=B)
    fill_llama(m, SEED)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, m.cfg.vocab, size=n).tolist() for n in (3, 9, 1, 5)]
    us = rng.random((steps, B)).astype(np.float32)
    first = [11, 22, 33, 44]

    def prompt():
        m.reset()
        for b, p in enumerate(prompts):
            m.prefill(p, seq=b)

    prompt()
    out = ctx.alloc(4 * steps * B)
    m.decode_sample_batch(first, steps, SETTINGS, ctx.to_device(us), out)
    got = out.download(np.int32).reshape(steps, B)
    assert [m.seq_position(b) for b in range(B)] == [len(p) + steps for p in prompts]

    prompt()
    lg, toks = ctx.alloc(4 * B * m.cfg.vocab), first
    for s in range(steps):
        m.forward_batch(toks, lg)
        x = lg.download(np.float32).reshape(B, -1)
        toks = [R.sample(x[b], *SETTINGS[b], us[s, b])[0] for b in range(B)]
        assert got[s].tolist() == toks, s
    m.close()


def test_group_of_one_gathers_the_logits():
    """A one-rank group takes the sharded path: the vocabulary's shards gathered, then sampled, alone
    and as a batch, and its captured steps go before the group."""
    with Context(0) as c:
        c.tp_init(1, 0, c.tp_unique_id())
        test_decode_sample_matches_sampling_the_logits(c)
        test_decode_sample_batch(c)


def test_refusals(ctx):
    m = Llama(ctx, _cfg(max_seq=4))
    fill_llama(m, SEED)
    u, out = ctx.to_device(np.zeros(8, np.float32)), ctx.alloc(64)
    for args, status in (((9999, 2, SETTINGS[0], u, out), -1), ((1, 0, SETTINGS[0], u, out), -1),
                         ((1, 5, SETTINGS[0], u, out), -8), ((1, 2**31 - 1, SETTINGS[0], u, out), -8),
                         ((1, 2, SETTINGS[0], int(u) + 2, out), -3)):
        with pytest.raises(MLMError) as e:
            m.decode_sample(*args)
        assert e.value.status == status and "mlm_llama_decode_sample" in str(e.value)
    assert m.position == 0
    assert ctx.lib.mlm_llama_decode_sample(m.handle, 1, 2, None, int(u), int(out)) == -1
    assert ctx.lib.mlm_llama_decode_sample_batch(m.handle, None, 2, None, int(u), int(out)) == -1
    with pytest.raises(ValueError):
        m.decode_sample_batch([1], 2, SETTINGS, u, out)
    m.close()
