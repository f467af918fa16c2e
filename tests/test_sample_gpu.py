"""Token sampling on the GPU against the plain 64-bit form: equal tokens."""
from __future__ import annotations

import numpy as np
import pytest

from metallm_b200 import MLMError, sample_params
from tests import kv4_reference as R

pytestmark = pytest.mark.gpu


def _run(ctx, x, params, u, stride=None):
    x = np.asarray(x, dtype=np.float32)
    rows, n = x.shape
    stride = stride or n
    wide = np.full((rows, stride), 1e30, np.float32)  # the padding between rows must not be read
    wide[:, :n] = x
    tok = ctx.to_device(np.full(rows, -7, np.int32))
    prob = ctx.to_device(np.full(rows, -7, np.float32))
    d, p, du = ctx.to_device(wide), ctx.to_device(sample_params(params)), ctx.to_device(np.asarray(u, np.float32))
    ctx.sample_f32(d, rows, n, stride, p, du, tok, prob)
    ctx.wait()
    return tok.download(np.int32, rows), prob.download(np.float32, rows)


def _check(ctx, x, params, u, stride=None):
    tok, prob = _run(ctx, x, params, u, stride)
    for r in range(len(x)):
        with np.errstate(all="ignore"):
            t, p = R.sample(x[r], *params[r], u[r])
        # the probability is one fp32 rounding of a 64-bit quotient
        assert tok[r] == t and abs(prob[r] - p) <= 2.0 ** -23 * p, (r, params[r], u[r], tok[r], t, prob[r], p)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.05), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 0.99, 0.0),
            (0.3, 0, 0.5, 0.0), (1.0, 0, 1.0, 0.1), (1.0, 1000, 0.99, 0.0), (0.0, 5, 0.5, 0.0), (1.0, 1, 1.0, 0.0),
            (2.0, 7, 0.0, 0.0), (1.0, 0, 1e-9, 0.0), (0.01, 0, 0.9, 0.0), (50.0, 300, 0.9, 0.0),
            (1.0, 20, 0.9, 2.0), (float("nan"), 0, 1.0, 0.0), (1.0, 0, float("nan"), float("nan")),
            (float("inf"), 0, 0.5, 0.0), (1e-30, 0, 0.9, 0.0), (-1.0, 0, 1.0, 0.0), (1.0, -3, 1.5, -1.0),
            (1.0, 2**31 - 1, 0.7, 0.0)]


@pytest.mark.parametrize("n", [1, 2, 31, 33, 500, 1000, 2047, 4099, 16385, 50257, 128256])
def test_settings(ctx, n):
    rng = np.random.default_rng(n)
    rows = len(SETTINGS)
    x = (2.2 * rng.standard_normal((rows, n)) - 3).astype(np.float32)
    for r in range(rows):
        x[r, rng.integers(0, n, 12)] += rng.uniform(0, 12, 12).astype(np.float32)
    _check(ctx, x, SETTINGS, rng.random(rows).astype(np.float32))


@pytest.mark.parametrize("rows", [1, 2, 5, 9, 18, 19, 37, 75, 149, 300])
def test_row_counts_and_strides(ctx, rows):
    """Every cluster size; rows at odd strides."""
    rng = np.random.default_rng(rows)
    n = 9001
    x = (3 * rng.standard_normal((rows, n))).astype(np.float32)
    params = [SETTINGS[r % 8] for r in range(rows)]
    _check(ctx, x, params, rng.random(rows).astype(np.float32), stride=n + 3)


@pytest.mark.parametrize("u", [0.0, 1e-30, 2.0**-24, 0.5, 1 - 2.0**-24, 1.0, 7.0, -1.0, float("nan")])
def test_uniform_edges(ctx, u):
    rng = np.random.default_rng(3)
    x = (2 * rng.standard_normal((4, 3000))).astype(np.float32)
    _check(ctx, x, SETTINGS[:4], [u] * 4)


@pytest.mark.parametrize("n", [5, 1025, 5000, 40000])
def test_ties(ctx, n):
    """Equal logits go by index: constant rows, a few levels, -0 beside +0; cuts inside the ties."""
    rng = np.random.default_rng(n)
    levels = rng.integers(0, 3, n).astype(np.float32)
    zeros = np.where(rng.random(n) < 0.5, np.float32(0), np.float32(-0.0))
    params, x = [], []
    for row in (np.full(n, -1.25, np.float32), levels, zeros):
        for p in ((1.0, 0, 1.0, 0.0), (1.0, max(1, n // 3), 1.0, 0.0), (1.0, 0, 0.37, 0.0), (1.0, n // 2 + 1, 0.7, 0.0),
                  (1.0, 0, 0.9, 0.5)):
            x.append(row)
            params.append(p)
    _check(ctx, np.stack(x), params, rng.random(len(x)).astype(np.float32))


def test_infinities_and_nan(ctx):
    n = 3001
    rng = np.random.default_rng(1)
    base = rng.standard_normal(n).astype(np.float32)
    nan, inf = np.float32(np.nan), np.float32(np.inf)
    some = base.copy()
    some[::3] = nan
    some[1::7] = -inf
    plus = base.copy()
    plus[[10, 2000, 2900]] = inf
    plus[5] = nan
    few = np.full(n, -inf, np.float32)
    few[[17, 1800]] = [1, 2]
    low = np.full(n, np.finfo(np.float32).min, np.float32)
    low[77] = 0
    x, params = [], []
    for row in (some, plus, few, low, np.full(n, nan), np.full(n, -inf), np.where(np.arange(n) < 9, nan, -inf),
                np.full(n, np.finfo(np.float32).min), np.linspace(-3e38, 3e38, n)):
        for p in SETTINGS[:8] + [(float("inf"), 0, 1.0, 0.0), (1.0, 5, 1.0, 0.0)]:
            x.append(np.asarray(row, np.float32))
            params.append(p)
    _check(ctx, np.stack(x), params, rng.random(len(x)).astype(np.float32))


def test_wide_rows_that_do_not_fit_shared_memory(ctx):
    rng = np.random.default_rng(12)
    n = (1 << 20) + 13
    x = (2 * rng.standard_normal((3, n))).astype(np.float32)
    _check(ctx, x, [(1.0, 0, 0.95, 0.0), (0.9, 3000, 1.0, 0.0), (1.0, 0, 1.0, 0.0)], [0.3, 0.8, 0.99])


def test_draws_follow_the_distribution(ctx):
    """The same row under evenly spread numbers: each token as often as its weight says."""
    rng = np.random.default_rng(2)
    rows, n = 2000, 64
    x = np.tile(rng.standard_normal(n).astype(np.float32), (rows, 1))
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    tok, _ = _run(ctx, x, [(1.0, 0, 1.0, 0.0)] * rows, u)
    w = np.exp(x[0].astype(np.float64))
    # a token's share of an even grid is within one step of its weight
    assert np.all(np.abs(np.bincount(tok, minlength=n) - rows * w / w.sum()) <= 1.01)


def test_graph_replay_and_no_prob(ctx):
    """Captured once, replayed with new logits, settings and numbers in the same buffers."""
    rng = np.random.default_rng(4)
    rows, n = 3, 5000
    d, p, u = ctx.alloc(4 * rows * n), ctx.alloc(16 * rows), ctx.alloc(4 * rows)
    tok = ctx.alloc(4 * rows)
    ctx.wait()
    ctx.graph_begin()
    ctx.sample_f32(d, rows, n, n, p, u, tok)
    g = ctx.graph_end()
    for step in range(4):
        x = (2 * rng.standard_normal((rows, n))).astype(np.float32)
        params = [SETTINGS[(step * rows + r) % 8] for r in range(rows)]
        us = rng.random(rows).astype(np.float32)
        d.upload(x)
        p.upload(sample_params(params))
        u.upload(us)
        g.launch()
        ctx.wait()
        want = [R.sample(x[r], *params[r], us[r])[0] for r in range(rows)]
        assert tok.download(np.int32, rows).tolist() == want
    g.destroy()


def test_refusals(ctx):
    b = ctx.alloc(1024)
    for args, status in (((b, 0, 4, 4, b, b, b), -2), ((b, 1, 0, 4, b, b, b), -2), ((b, 1, (1 << 22) + 1, 1 << 23, b, b, b), -2),
                         ((b, 2, 8, 7, b, b, b), -2), ((b, 1, 4, 4, None, b, b), -1), ((int(b) + 2, 1, 4, 4, b, b, b), -3)):
        with pytest.raises(MLMError) as e:
            ctx.sample_f32(*args)
        assert e.value.status == status and "mlm_sample_f32" in str(e.value)
