"""The 4-bit KV cache on the GPU: quantizing append, read-back, attention."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from metallm_b200 import (TYPE_BF16, TYPE_F16, TYPE_F32, Kv4Cache, MLMError)
from tests import kv4_reference as R

pytestmark = pytest.mark.gpu

FILL = 0xA5


def _bf16(x):
    """fp32 values rounded to bf16 (nearest even), as fp32 and as uint16 bits."""
    b = np.asarray(x, dtype=np.float32).view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return (r.astype(np.uint32) << 16).view(np.float32), r


def _cache(ctx, batch, n_kv, capacity):
    c = ctx.kv4_cache(batch, n_kv, capacity)
    for p in (c.k_buffer, c.v_buffer):
        ctx.call("mlm_memset", p, FILL, p.nbytes)
    return c


def _rows(buf, batch, n_kv, capacity):
    return buf.download(np.uint8, batch * n_kv * capacity * R.ROW).reshape(batch, n_kv, capacity, R.ROW)


def _ints(ctx, v):
    return ctx.to_device(np.asarray(v, dtype=np.int32))


def _inputs(rng, shape, kind):
    x = rng.standard_normal(shape).astype(np.float32)
    x[..., 3::37] *= 20
    if kind == "edges":  # constant groups, zeros, tiny and huge values, a whole group at the limits
        x[..., :32] = 1.7
        x[..., 32:64] = 0
        x[..., 64:96] *= 1e-7
        x[..., 96:100] = [7e4, -7e4, 65504, -65504]
    return x


@pytest.mark.parametrize("batch,n_kv,tokens,capacity,type,pad,ragged", [
    (1, 8, 1, 64, TYPE_F32, 4096 + 1024, False),
    (1, 1, 1, 1, TYPE_F16, 0, False),
    (3, 2, 7, 11, TYPE_BF16, 0, True),
    (2, 5, 33, 40, TYPE_F32, 4, True),
    (4, 3, 17, 17, TYPE_F16, 8, False),
    (1, 16, 300, 513, TYPE_F32, 0, False),
    (70, 1, 2, 9, TYPE_F16, 0, True),
])
@pytest.mark.parametrize("kind", ["normal", "edges"])
def test_append_and_read(ctx, batch, n_kv, tokens, capacity, type, pad, ragged, kind):
    rng = np.random.default_rng(tokens * 7 + batch)
    stride = n_kv * R.D + pad
    src, dev = [], []
    for _ in "kv":
        x = _inputs(rng, (batch, tokens, stride), "normal")
        x[..., :n_kv * R.D] = _inputs(rng, (batch, tokens, n_kv, R.D), kind).reshape(batch, tokens, -1)
        if type == TYPE_F16:
            with np.errstate(over="ignore"):
                x = x.astype(np.float16)
            dev.append(ctx.to_device(x))
        elif type == TYPE_BF16:
            x, bits = _bf16(x)
            dev.append(ctx.to_device(bits))
        else:
            dev.append(ctx.to_device(x))
        src.append(np.asarray(x, dtype=np.float32)[..., :n_kv * R.D].reshape(batch, tokens, n_kv, R.D))
    counts = [tokens - (b * 3) % (tokens + 1) for b in range(batch)] if ragged else [tokens] * batch
    pos = [(b * 5) % (capacity - tokens + 1) for b in range(batch)]
    c = _cache(ctx, batch, n_kv, capacity)
    cnt = _ints(ctx, counts) if ragged else None
    ctx.kv4_append(c, dev[0], dev[1], type, stride, tokens, _ints(ctx, pos), cnt)
    outs = [ctx.to_device(np.full(batch * tokens * n_kv * R.D, 7, np.float16)) for _ in "kv"]
    ctx.kv4_read_f16(c, tokens, _ints(ctx, pos), cnt, *outs)
    ctx.wait()
    for x, buf, out in zip(src, (c.k_buffer, c.v_buffer), outs):
        want = np.full((batch, n_kv, capacity, R.ROW), FILL, np.uint8)
        back = np.full((batch, tokens, n_kv, R.D), 7, np.float16)
        q = R.quantize(x)
        for b in range(batch):
            want[b, :, pos[b]:pos[b] + counts[b]] = q[b, :counts[b]].transpose(1, 0, 2)
            # m + d c has at most 22 bits above 2^-24: one 32-bit rounding, then the fp16 one
            back[b, :counts[b]] = R.values(q[b, :counts[b]]).astype(np.float32).astype(np.float16)
        assert np.array_equal(_rows(buf, batch, n_kv, capacity), want)
        got = out.download(np.float16).reshape(back.shape)
        assert np.all(np.isfinite(got)) and np.array_equal(got, back)


def test_append_nan_marks_its_group_alone(ctx):
    x = np.ones((1, 1, 1, R.D), np.float32) * np.arange(R.D, dtype=np.float32)
    x[..., 40] = np.nan
    x[..., 70] = np.inf
    c = _cache(ctx, 1, 1, 2)
    dev = ctx.to_device(x)
    ctx.kv4_append(c, dev, dev, TYPE_F32, R.D, 1, _ints(ctx, [1]))
    outs = [ctx.alloc(256) for _ in "kv"]
    ctx.kv4_read_f16(c, 1, _ints(ctx, [1]), None, *outs)
    got = outs[0].download(np.float16)
    assert np.all(np.isnan(got[32:64])) and np.all(np.isfinite(np.delete(got, np.s_[32:64])))
    assert got[70] > 60000
    assert np.all(_rows(c.v_buffer, 1, 1, 2)[0, 0, 0] == FILL)


@pytest.mark.parametrize("pos,counts", [([3, 0], None), ([-1, 2], None), ([0, 0], [3, 1]), ([0, 0], [-1, 2]),
                                        ([2**31 - 1, 0], None), ([-2**31, 0], None)])
def test_append_outside_the_cache_is_skipped_and_reported(ctx, pos, counts):
    batch, n_kv, tokens, capacity = 2, 3, 2, 4
    x = np.random.default_rng(1).standard_normal((batch, tokens, n_kv, R.D)).astype(np.float32)
    c = _cache(ctx, batch, n_kv, capacity)
    dev = ctx.to_device(x)
    ctx.kv4_append(c, dev, dev, TYPE_F32, n_kv * R.D, tokens, _ints(ctx, pos),
                   None if counts is None else _ints(ctx, counts))
    with pytest.raises(MLMError) as e:
        ctx.wait()
    assert e.value.status == -2 and "outside its cache" in str(e.value)
    ctx.wait()  # reported once
    want = np.full((batch, n_kv, capacity, R.ROW), FILL, np.uint8)
    q = R.quantize(x)
    for b in range(batch):
        for t in range(min(tokens, tokens if counts is None else counts[b])):
            if 0 <= pos[b] + t < capacity:
                want[b, :, pos[b] + t] = q[b, t]
    assert np.array_equal(_rows(c.k_buffer, batch, n_kv, capacity), want)


def _attention_case(ctx, batch, tokens, n_heads, n_kv, lens, counts, out_type, capacity=None, seed=0,
                    spoil=True, q_scale=1.5, v_scale=None):
    """Runs mlm_attn_kv4 and compares it with the 64-bit form.  `spoil`: rows past a sequence's
    length hold NaN scales.  `v_scale`: factors of V per position."""
    rng = np.random.default_rng(seed + 1000 * tokens + batch)
    capacity = capacity or max(max(lens), 1)
    rows = []
    for name in "kv":
        x = rng.standard_normal((batch, n_kv, capacity, R.D)).astype(np.float32)
        x[..., 5::61] *= 4
        if name == "v" and v_scale is not None:
            x *= v_scale(np.arange(capacity, dtype=np.float32))[:, None]
        r = R.quantize(x)
        if spoil:
            for b in range(batch):
                r[b, :, max(lens[b], 0):] = 0xFF
        rows.append(r)
    q = (q_scale * rng.standard_normal((batch, tokens, n_heads, R.D))).astype(np.float16)
    dk, dv = (ctx.to_device(r) for r in rows)
    cache = Kv4Cache(int(dk), int(dv), batch, n_kv, R.D, capacity)
    fill = np.float16(77)
    shape = (batch, tokens, n_heads, R.D)
    out = ctx.to_device(np.full(shape, fill, np.float16) if out_type == TYPE_F16
                        else np.full(shape, 0x429A, np.uint16))
    full = counts if counts is not None else [tokens] * batch
    ctx.attn_kv4(cache, ctx.to_device(q), n_heads, tokens, _ints(ctx, lens),
                 None if counts is None else _ints(ctx, counts), out, out_type)
    ctx.wait()
    raw = out.download(np.uint16, int(np.prod(shape))).reshape(shape)
    got = (raw.view(np.float16).astype(np.float64) if out_type == TYPE_F16
           else (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64))
    ref, smax, vmax = R.attention(q, *rows, lens, full)
    live = ~np.isnan(ref[..., 0])
    assert np.all(got[~live] == 77)  # rows behind the last token are left as they were
    assert np.all(np.isfinite(got[live]))
    eps = 2.0 ** -10 if out_type == TYPE_F16 else 2.0 ** -7
    rounded = tokens * (n_heads // n_kv) > 16 and out_type != TYPE_F16
    few = tokens * (n_heads // n_kv) <= 16
    tol = R.attention_tolerance(ref, smax, vmax, eps, rounded, few and out_type != TYPE_F16)
    bad = np.abs(got - ref) > tol
    assert not np.any(bad[live]), (np.argwhere(bad & live[..., None])[:5], np.abs(got - ref)[live].max())
    a, r = got[live], ref[live]
    if np.linalg.norm(r) > 0:
        # half a step of rounding is at most eps/2, uniform: eps/2/sqrt(3) in the mean square; scores
        # and weights in 32 bits add little, operands rounded to fp16 (K, weights, V) 2^-11/sqrt(3)
        # each, K's and V's grown by the scores' spread (at most 4 here)
        bound = eps / 2 / 3 ** .5 + 3e-5 + (9 * 2.0 ** -11 / 3 ** .5 if rounded else 0)
        assert np.linalg.norm(a - r) / np.linalg.norm(r) < bound
    return got


@pytest.mark.parametrize("n_heads,n_kv", [(32, 8), (64, 8), (8, 8), (3, 1), (16, 1), (40, 8), (14, 2), (20, 1)])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 33, 64, 100, 255, 1025])
def test_decode_lengths(ctx, n_heads, n_kv, length):
    _attention_case(ctx, 1, 1, n_heads, n_kv, [length], None, TYPE_F16, capacity=length + 5)


@pytest.mark.parametrize("tokens,n_heads", [(1, 4), (1, 12), (5, 4), (9, 4)])
@pytest.mark.parametrize("v_scale", ["one", "small", "large", "mixed"])
def test_long_cache_keeps_the_small_weights(ctx, tokens, n_heads, v_scale):
    """Many rows of little weight each, whose sum nearly cancels: the weights need more bits than the
    largest one's fp16 step, whatever V's scale, and where V grows on the way."""
    scale = {"one": lambda j: 1 + 0 * j, "small": lambda j: 0.02 + 0 * j, "large": lambda j: 3000 + 0 * j,
             "mixed": lambda j: np.where(j % 997 == 500, 40, 1).astype(np.float32)}[v_scale]
    _attention_case(ctx, 1, tokens, n_heads, 1, [60001], None, TYPE_F16, capacity=60010, v_scale=scale)


@pytest.mark.parametrize("out_type", [TYPE_F16, TYPE_BF16])
def test_many_long_caches(ctx, out_type):
    """Long stretches of one cache in the same accumulators: 128 sequences (the same rows, their own
    queries), the outputs' two halves (codes and minima) nearly cancelling."""
    rng = np.random.default_rng(12)
    batch, n_heads, n = 128, 4, 32768
    rows = [R.quantize(rng.standard_normal((1, 1, n, R.D)).astype(np.float32)) for _ in "kv"]
    q = (1.5 * rng.standard_normal((batch, 1, n_heads, R.D))).astype(np.float16)
    dk, dv = (ctx.to_device(np.repeat(r, batch, axis=0)) for r in rows)
    out = ctx.alloc(2 * q.size)
    ctx.attn_kv4(Kv4Cache(int(dk), int(dv), batch, 1, R.D, n), ctx.to_device(q), n_heads, 1,
                 _ints(ctx, [n] * batch), None, out, out_type)
    ctx.wait()
    raw = out.download(np.uint16).reshape(q.shape)
    got = (raw.view(np.float16).astype(np.float64) if out_type == TYPE_F16
           else (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64))
    eps = 2.0 ** -10 if out_type == TYPE_F16 else 2.0 ** -7
    for b in (0, 61, 127):
        ref = R.attention(q[b:b + 1], *rows, [n], [1])[0][0]
        # half a step of rounding, uniform: eps / 2 / sqrt(3) in the mean square; a bf16 output's
        # weights are fp16 products p d, twice rounded (2^-11 / sqrt(3) each) against codes that are
        # not centred (their mean square at most 2.5 of the values')
        bound = eps / 2 / 3 ** .5 + 3e-5 + (0 if out_type == TYPE_F16 else 2.5 * 2 ** .5 * 2.0 ** -11 / 3 ** .5)
        assert np.linalg.norm(got[b] - ref) / np.linalg.norm(ref) < bound


@pytest.mark.parametrize("out_type", [TYPE_F16, TYPE_BF16])
@pytest.mark.parametrize("lens", [[0], [0, 0, 0], [5, 0, 700, 1, 64, 0, 333], [2000, 1], [0, 4000],
                                  list(range(40))])
def test_decode_ragged(ctx, lens, out_type):
    _attention_case(ctx, len(lens), 1, 8, 2, lens, None, out_type, capacity=max(lens) + 3)


def test_decode_many_sequences(ctx):
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 60, 1024).tolist()
    _attention_case(ctx, 1024, 1, 4, 1, lens, None, TYPE_F16, capacity=64)


def test_decode_long(ctx):
    _attention_case(ctx, 2, 1, 8, 2, [30011, 12345], None, TYPE_F16, capacity=30016)


@pytest.mark.parametrize("tokens,n_heads,n_kv", [(2, 8, 8), (4, 8, 2), (3, 32, 8), (5, 4, 2), (8, 8, 8), (16, 2, 2),
                                                 (2, 8, 1), (7, 7, 7)])
@pytest.mark.parametrize("out_type", [TYPE_F16, TYPE_BF16])
def test_few_tokens(ctx, tokens, n_heads, n_kv, out_type):
    lens = [tokens, 0, tokens - 1, 130, 517]
    _attention_case(ctx, 5, tokens, n_heads, n_kv, lens, None, out_type, capacity=520)
    counts = [tokens, 1, 0, tokens // 2, tokens - 1]
    _attention_case(ctx, 5, tokens, n_heads, n_kv, lens, counts, out_type, capacity=520, seed=1)


@pytest.mark.parametrize("tokens,n_heads,n_kv", [(17, 4, 4), (33, 8, 2), (64, 4, 1), (100, 8, 1), (20, 14, 2),
                                                 (130, 3, 1)])
@pytest.mark.parametrize("out_type", [TYPE_F16, TYPE_BF16])
def test_prompt_chunks(ctx, tokens, n_heads, n_kv, out_type):
    lens = [tokens, tokens + 1, 300, 5, 0]
    _attention_case(ctx, 5, tokens, n_heads, n_kv, lens, None, out_type, capacity=301)
    counts = [tokens, 1, tokens - 3, 5, 0]
    _attention_case(ctx, 5, tokens, n_heads, n_kv, lens, counts, out_type, capacity=301, seed=1)


def test_prompt_of_many_tokens(ctx):
    _attention_case(ctx, 1, 513, 4, 2, [900], None, TYPE_BF16)


@pytest.mark.parametrize("tokens", [1, 3, 40])
@pytest.mark.parametrize("q_scale", [0.0, 1e-4, 60.0])
def test_sharp_and_flat_scores(ctx, tokens, q_scale):
    """Zero queries average V; large ones pick single keys (scores in the hundreds)."""
    rng = np.random.default_rng(9)
    batch, n_kv, n_heads, n = 1, 2, 8, 200
    rows = [R.quantize(rng.standard_normal((batch, n_kv, n, R.D)).astype(np.float32)) for _ in "kv"]
    q = (q_scale * rng.standard_normal((batch, tokens, n_heads, R.D))).astype(np.float16)
    dk, dv = (ctx.to_device(r) for r in rows)
    out = ctx.alloc(2 * q.size)
    ctx.attn_kv4(Kv4Cache(int(dk), int(dv), batch, n_kv, R.D, n), ctx.to_device(q), n_heads, tokens,
                 _ints(ctx, [n]), None, out, TYPE_F16)
    ctx.wait()
    ref, smax, vmax = R.attention(q, *rows, [n], [tokens])
    got = out.download(np.float16).reshape(q.shape).astype(np.float64)
    tol = R.attention_tolerance(ref, smax, vmax, 2.0 ** -10, tokens * 4 > 16)
    assert np.all(np.abs(got - ref) <= tol)


def test_nan_key_reaches_only_tokens_that_see_it(ctx):
    """A NaN key of a later token must not reach an earlier one through the shared tile."""
    for tokens, n in ((4, 40), (40, 100)):
        rng = np.random.default_rng(2)
        rows = [R.quantize(rng.standard_normal((1, 1, n, R.D)).astype(np.float32)) for _ in "kv"]
        for r in rows:
            r[0, 0, n - 1, 64:] = 0xFF  # the last token's own row
        q = rng.standard_normal((1, tokens, 2, R.D)).astype(np.float16)
        dk, dv = (ctx.to_device(r) for r in rows)
        out = ctx.alloc(2 * q.size)
        ctx.attn_kv4(Kv4Cache(int(dk), int(dv), 1, 1, R.D, n), ctx.to_device(q), 2, tokens,
                     _ints(ctx, [n]), None, out, TYPE_F16)
        ctx.wait()
        got = out.download(np.float16).reshape(q.shape)
        assert np.all(np.isfinite(got[0, :-1])) and np.all(np.isnan(got[0, -1]))


@pytest.mark.parametrize("lens,counts,seen", [([9, 3], None, [6, 3]), ([-4, 3], None, [0, 3]), ([2**31 - 1, 1], None, [6, 1]),
                                              ([4, 3], [2, 1], [4, 3])])
def test_attention_lengths_outside_the_cache_are_kept_within(ctx, lens, counts, seen):
    rng = np.random.default_rng(3)
    rows = [R.quantize(rng.standard_normal((2, 1, 6, R.D)).astype(np.float32)) for _ in "kv"]
    q = rng.standard_normal((2, 1, 2, R.D)).astype(np.float16)
    dk, dv = (ctx.to_device(r) for r in rows)
    out = ctx.alloc(2 * q.size)
    ctx.attn_kv4(Kv4Cache(int(dk), int(dv), 2, 1, R.D, 6), ctx.to_device(q), 2, 1, _ints(ctx, lens),
                 None if counts is None else _ints(ctx, counts), out, TYPE_F16)
    with pytest.raises(MLMError) as e:
        ctx.wait()
    assert e.value.status == -2
    ref, smax, vmax = R.attention(q, *rows, seen, [1, 1])
    got = out.download(np.float16).reshape(q.shape).astype(np.float64)
    assert np.all(np.abs(got - ref) <= R.attention_tolerance(ref, smax, vmax, 2.0 ** -10, False))


def test_cache_past_32_bit_offsets(ctx):
    """A cache of more than 2^32 bytes: its last rows, by append, read and attention."""
    n_kv, capacity = 8, (2**32 // (8 * R.ROW)) + 70000
    import torch
    if torch.cuda.mem_get_info(ctx.device)[0] < 12 * 2**30:
        pytest.skip("not enough free memory")
    c = ctx.kv4_cache(1, n_kv, capacity)
    try:
        n = 65
        rng = np.random.default_rng(4)
        x = rng.standard_normal((1, n, n_kv, R.D)).astype(np.float32)
        dev = ctx.to_device(x)
        pos = _ints(ctx, [capacity - n])
        ctx.kv4_append(c, dev, dev, TYPE_F32, n_kv * R.D, n, pos)
        outs = [ctx.alloc(2 * x.size) for _ in "kv"]
        ctx.kv4_read_f16(c, n, pos, None, *outs)
        ctx.wait()
        want = R.values(R.quantize(x)).astype(np.float32).astype(np.float16)
        for o in outs:
            assert np.array_equal(o.download(np.float16).reshape(want.shape), want)
        # rows of the last head end at the cache's end: attend to them through a view whose
        # first row is the tail's
        tail = (n_kv * capacity - n) * R.ROW
        view = Kv4Cache(c.k + tail, c.v + tail, 1, 1, R.D, n)
        q = rng.standard_normal((1, 1, 4, R.D)).astype(np.float16)
        out = ctx.alloc(2 * q.size)
        ctx.attn_kv4(view, ctx.to_device(q), 4, 1, _ints(ctx, [n]), None, out, TYPE_F16)
        ctx.wait()
        rows = R.quantize(x[:, :, -1:]).transpose(0, 2, 1, 3)
        ref, smax, vmax = R.attention(q, rows, rows, [n], [1])
        got = out.download(np.float16).reshape(q.shape).astype(np.float64)
        assert np.all(np.abs(got - ref) <= R.attention_tolerance(ref, smax, vmax, 2.0 ** -10, False))
    finally:
        c.free()


def test_results_do_not_depend_on_the_run(ctx):
    """The same call twice gives the same bits (no order of arrival in the sums)."""
    rng = np.random.default_rng(6)
    for batch, tokens, n in ((3, 1, 9000), (2, 60, 1500)):
        rows = [R.quantize(rng.standard_normal((batch, 2, n, R.D)).astype(np.float32)) for _ in "kv"]
        q = rng.standard_normal((batch, tokens, 8, R.D)).astype(np.float16)
        dk, dv = (ctx.to_device(r) for r in rows)
        cache, dq, dl = Kv4Cache(int(dk), int(dv), batch, 2, R.D, n), ctx.to_device(q), _ints(ctx, [n] * batch)
        got = []
        for _ in range(4):
            out = ctx.alloc(2 * q.size)
            ctx.attn_kv4(cache, dq, 8, tokens, dl, None, out, TYPE_F16)
            ctx.wait()
            got.append(out.download(np.uint16))
        assert all(np.array_equal(got[0], g) for g in got[1:])


def test_append_attend_read_in_a_replayed_graph(ctx):
    """A decode loop as a user runs it: append and attend captured once and replayed
    while the positions in device memory grow; each step equals the plain form."""
    batch, n_kv, n_heads, capacity, steps = 3, 2, 8, 40, 25
    rng = np.random.default_rng(8)
    c = _cache(ctx, batch, n_kv, capacity)
    kv = [ctx.alloc(4 * batch * n_kv * R.D) for _ in "kv"]
    q = ctx.alloc(2 * batch * n_heads * R.D)
    pos, lens, out = _ints(ctx, [0] * batch), _ints(ctx, [0] * batch), ctx.alloc(2 * batch * n_heads * R.D)
    ctx.wait()
    ctx.graph_begin()
    ctx.kv4_append(c, kv[0], kv[1], TYPE_F32, n_kv * R.D, 1, pos)
    ctx.attn_kv4(c, q, n_heads, 1, lens, None, out, TYPE_F16)
    g = ctx.graph_end()
    hist = [np.zeros((batch, n_kv, capacity, R.ROW), np.uint8) for _ in "kv"]
    start = np.array([0, 7, 15])
    for h, buf in zip(hist, (c.k_buffer, c.v_buffer)):  # rows that were there before
        for b in range(batch):
            h[b, :, :start[b]] = R.quantize(rng.standard_normal((n_kv, start[b], R.D)))
        buf.upload(h)
    for s in range(steps):
        at = (start + s).astype(np.int32)
        x = [rng.standard_normal((batch, n_kv, R.D)).astype(np.float32) for _ in "kv"]
        qs = rng.standard_normal((batch, 1, n_heads, R.D)).astype(np.float16)
        for d, v in zip(kv, x):
            d.upload(v)
        q.upload(qs)
        pos.upload(at)
        lens.upload(at + 1)
        g.launch()
        ctx.wait()
        for h, v in zip(hist, x):
            for b in range(batch):
                h[b, :, at[b]] = R.quantize(v[b])
        ref, smax, vmax = R.attention(qs, *hist, (at + 1).tolist(), [1] * batch)
        got = out.download(np.float16).reshape(qs.shape).astype(np.float64)
        assert np.all(np.abs(got - ref) <= R.attention_tolerance(ref, smax, vmax, 2.0 ** -10, False))
    g.destroy()


def test_calls_on_another_stream(ctx):
    """The ops follow mlm_set_stream: work queued there before them is seen."""
    import torch
    s = torch.cuda.Stream()
    rng = np.random.default_rng(11)
    n = 300
    x = rng.standard_normal((1, n, 2, R.D)).astype(np.float32)
    q = rng.standard_normal((1, 1, 4, R.D)).astype(np.float16)
    host = torch.from_numpy(x).pin_memory()
    ctx.set_stream(s.cuda_stream)
    try:
        with torch.cuda.stream(s):
            dev = torch.zeros(x.shape, device="cuda")
            big = torch.randn(4096, 4096, device="cuda")
            for _ in range(4):
                big = big @ big * 1e-3
            dev.copy_(host, non_blocking=True)
        c = ctx.kv4_cache(1, 2, n)
        out = ctx.alloc(2 * q.size)
        dq, dl, dp = ctx.to_device(q), _ints(ctx, [n]), _ints(ctx, [0])
        ctx.kv4_append(c, dev.data_ptr(), dev.data_ptr(), TYPE_F32, 2 * R.D, n, dp)
        ctx.attn_kv4(c, dq, 4, 1, dl, None, out, TYPE_F16)
        ctx.wait()
        rows = R.quantize(x).transpose(0, 2, 1, 3)
        ref, smax, vmax = R.attention(q, rows, rows, [n], [1])
        got = out.download(np.float16).reshape(q.shape).astype(np.float64)
        assert np.all(np.abs(got - ref) <= R.attention_tolerance(ref, smax, vmax, 2.0 ** -10, False))
    finally:
        ctx.set_stream(0)


def test_refusals_name_the_call(ctx):
    c = ctx.kv4_cache(2, 2, 8)
    b = ctx.alloc(1 << 16)
    p = _ints(ctx, [0, 0])
    with pytest.raises(MLMError) as e:
        ctx.kv4_append(c, b, b, TYPE_F32, 2 * R.D, 9, p)
    assert e.value.status == -2 and "mlm_kv4_append" in str(e.value)
    with pytest.raises(MLMError) as e:
        ctx.attn_kv4(c, b, 3, 1, p, None, b, TYPE_F16)
    assert e.value.status == -2 and "mlm_attn_kv4" in str(e.value)
    with pytest.raises(MLMError) as e:
        ctx.attn_kv4(c, int(b) + 2, 2, 1, p, None, b, TYPE_F16)
    assert e.value.status == -3
    assert ctypes.sizeof(Kv4Cache) == 32
