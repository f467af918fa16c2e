"""Attention over the 4-bit cache where its precision is at stake: small weights beside large
ones, long stretches of a cache walked by one CTA, sharp scores."""
from __future__ import annotations

import numpy as np
import pytest

from metallm_b200 import TYPE_BF16, TYPE_F16, Kv4Cache
from tests import kv4_reference as R

pytestmark = pytest.mark.gpu


def _parts(rows):
    """m and d c of cache rows [..., 80], in 64 bits: [..., 128] each."""
    zero = rows.copy()
    zero[..., :64] = 0
    m = R.values(zero)
    return m, R.values(rows) - m


def _attend(ctx, k_rows, v_rows, batch, q, out_type):
    """q [batch][tokens][heads][128] over `batch` copies of one KV head's rows [n][80]."""
    import torch
    n = k_rows.shape[0]
    dk, dv = (torch.from_numpy(r).cuda().expand(batch, n, R.ROW).contiguous() for r in (k_rows, v_rows))
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    dq = torch.from_numpy(q).cuda()
    out = torch.zeros(q.shape, dtype=torch.float16 if out_type == TYPE_F16 else torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    ctx.attn_kv4(Kv4Cache(dk.data_ptr(), dv.data_ptr(), batch, 1, R.D, n), dq.data_ptr(), q.shape[2],
                 q.shape[1], lens.data_ptr(), None, out.data_ptr(), out_type)
    ctx.wait()
    return out.double().cpu().numpy()


# ---- small weights beside large ones -------------------------------------------

N_PEAKED, PERIOD = 32768, 8192
V_KINDS = {
    "one": lambda x, j: x,
    "small": lambda x, j: x * 0.002,
    # one group spans 30 and more, the others do not
    "wide": lambda x, j: np.concatenate([x[:, :96], x[:, 96:] * 60], 1),
    # single rows of 40 times the others' scale, in two groups
    "late": lambda x, j: np.where((j % 997 == 500)[:, None] & (np.arange(R.D) >= 64), x * 40, x),
}


@pytest.fixture(scope="module", params=list(V_KINDS))
def peaked(request):
    """Keys of which every 8192nd outweighs the others by as many octaves as the query says, and whose
    own value row is zero: the outputs are what the small weights add up to."""
    rng = np.random.default_rng(7)
    j = np.arange(N_PEAKED)
    k = 0.3 * rng.standard_normal((N_PEAKED, R.D)).astype(np.float32)
    v = (1 + 0.3 * rng.standard_normal((N_PEAKED, R.D))).astype(np.float32)
    v = V_KINDS[request.param](v, j).astype(np.float32)
    peak = j % PERIOD == 0
    k[:, 0] = np.where(peak, 8, 0)
    v[peak] = 0
    return R.quantize(k), R.quantize(v)


@pytest.mark.parametrize("out_type", [TYPE_F16, TYPE_BF16])
@pytest.mark.parametrize("heads", [4, 8, 16, 32])
def test_small_weights_beside_large_ones(ctx, peaked, heads, out_type):
    """1024 sequences, so that a warp walks thousands of rows behind a dominant key."""
    k_rows, v_rows = peaked
    rng = np.random.default_rng(heads)
    q = 0.05 * rng.standard_normal((1, 1, heads, R.D))
    q[0, 0, :, 0] = np.linspace(15.3, 25.6, heads) * np.log(2) * np.sqrt(R.D) / 8  # octaves
    q = q.astype(np.float16)
    batch = 1024
    got = _attend(ctx, k_rows, v_rows, batch, np.repeat(q, batch, axis=0), out_type)[:, 0]

    x = q[0, 0].astype(np.float64)
    k, (m, dc) = R.values(k_rows), _parts(v_rows)
    s = x @ k.T / np.sqrt(R.D)
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    ref = p @ (m + dc)
    # An error e of every score moves a weight by its expm1(e) at most, the sum of them too: 2 e of the
    # mean |v|.  A score's is 128 roundings of 2^-23 of sum |q k|; the many-row form to bf16 rounds K to
    # fp16, 2^-11 of it.  exp and the sums: 2^-18.
    many = heads > 16
    bf16 = out_type == TYPE_BF16
    smax = (np.abs(x) @ np.abs(k).T).max(1, keepdims=True) / np.sqrt(R.D)
    e = smax * (128 * 2.0 ** -23 + (2.0 ** -11 if many and bf16 else 0))
    mean_m, mean_dc = p @ np.abs(m), p @ np.abs(dc)
    tol = (np.expm1(2 * e) + 2.0 ** -18) * (mean_m + mean_dc)
    # to bf16 the weights are fp16 values (2^-11), then few rows' p d and many rows' V once more
    if bf16:
        tol += 2.0 ** -11 * (mean_m + 2 * mean_dc) * (1 + 2.0 ** -8) + (2.0 ** -11 * mean_m if many else 0)
    # a weight (and a p d, of the largest d) is held to 2^-25 where the largest weight is 2^10 or more; 2^7
    # or more with many rows
    vmax = (np.abs(m).reshape(-1, 4, 32) + 15 / 7.5 * np.abs(dc).reshape(-1, 4, 32)).max((0, 2)).repeat(32)
    tol += 2 * N_PEAKED * 2.0 ** (-32 if many else -35) * vmax
    tol += (2.0 ** -8 if bf16 else 2.0 ** -11) * (np.abs(ref) + tol) + 2.0 ** -25
    over = np.abs(got - ref) / tol
    at = np.unravel_index(over.argmax(), over.shape)
    assert over.max() <= 1, (at, got[at], ref[at[1:]], over.max())


# ---- long stretches walked by one CTA ---------------------------------------------

@pytest.mark.parametrize("keys", ["random", "flat"])
@pytest.mark.parametrize("out_type", [TYPE_F16, TYPE_BF16])
@pytest.mark.parametrize("tokens,heads", [(5, 4), (40, 4)])
def test_long_items_do_not_shrink(ctx, tokens, heads, out_type, keys):
    """More items of 1024 key tiles than SMs: one CTA sums most of an item.  What each addition
    cuts off (or rounds in one direction, where all weights are alike) must not add up."""
    rng = np.random.default_rng(tokens)
    batch, n = 160, 131072
    v = (1 + rng.random(R.D) + 0.3 * rng.standard_normal((n, R.D))).astype(np.float32)
    if keys == "random":
        k = rng.standard_normal((n, R.D)).astype(np.float32)
        q = 1.2 * rng.standard_normal((1, tokens, heads, R.D))
    else:  # one key above all the others, by a fraction of an octave
        k = np.repeat(rng.standard_normal((1, R.D)), n, axis=0).astype(np.float32)
        k[:, 0] = 0
        k[0, 0] = 8
        q = np.zeros((1, tokens, heads, R.D))
        q[..., 0] = rng.uniform(0.2, 0.9, (tokens, heads)) * np.log(2) * np.sqrt(R.D) / 8
    q = q.astype(np.float16)
    k_rows, v_rows = R.quantize(k), R.quantize(v)
    got = _attend(ctx, k_rows, v_rows, batch, np.repeat(q, batch, axis=0), out_type)

    kv, vv = R.values(k_rows), R.values(v_rows)
    ref = np.empty((tokens, heads, R.D))
    for t in range(tokens):
        s = q[0, t].astype(np.float64) @ kv[:n - tokens + t + 1].T / np.sqrt(R.D)
        p = np.exp(s - s.max(1, keepdims=True))
        ref[t] = p @ vv[:len(s[0])] / p.sum(1, keepdims=True)
    eps = 2.0 ** -10 if out_type == TYPE_F16 else 2.0 ** -7
    # half a step of rounding, uniform, in the mean square; operands rounded to fp16 for bf16 outputs
    bound = eps / 2 / 3 ** .5 + 3e-5 + (9 * 2.0 ** -11 / 3 ** .5 if out_type == TYPE_BF16 else 0)
    assert np.linalg.norm(got - ref) / (batch ** .5 * np.linalg.norm(ref)) < bound
    if out_type == TYPE_F16:
        # The mean over a head's outputs, whose own roundings cancel: four deviations of their mean.  A sum
        # of 128 key tiles takes 24 products each, every one cutting off at most 2^-23 of what is there,
        # half of the sum on average: 1.84e-4.
        bias = (got / ref - 1).mean((1, 3))  # [batch][heads]
        assert np.abs(bias).max() < 1.84e-4 + 4 * eps / 2 / 3 ** .5 / (tokens * R.D) ** .5


# ---- infinities in queries ----------------------------------------------------------

@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan, 65504.0])
@pytest.mark.parametrize("tokens,heads", [(2, 2), (4, 2), (8, 2), (20, 2)])
def test_a_token_that_sees_nothing_gives_zeros_whatever_its_query(ctx, tokens, heads, value):
    """Two rows cached: all but the last two tokens see none of them."""
    rng = np.random.default_rng(tokens)
    q = rng.standard_normal((1, tokens + 2, heads, R.D)).astype(np.float16)
    q[0, :tokens, 0, 5] = value
    k, v = (R.quantize(rng.standard_normal((2, R.D)).astype(np.float32)) for _ in "kv")
    got = _attend(ctx, k, v, 1, q, TYPE_F16)
    assert np.all(got[0, :tokens] == 0)
    assert np.all(np.isfinite(got[0, tokens:]))


# ---- sharp scores --------------------------------------------------------------------

@pytest.mark.parametrize("tokens,heads", [(3, 4), (2, 8), (4, 4), (40, 4)])
@pytest.mark.parametrize("out_type", [TYPE_F16, TYPE_BF16])
@pytest.mark.parametrize("q_scale", [0.0, 1e-4, 8.0, 60.0])
def test_sharp_and_flat_scores_to_their_own_precision(ctx, tokens, heads, out_type, q_scale):
    """Each output type against the operands that it takes: an fp16 output's are never rounded alone."""
    rng = np.random.default_rng(9)
    n = 200
    k, v = (R.quantize(rng.standard_normal((n, R.D)).astype(np.float32)) for _ in "kv")
    q = (q_scale * rng.standard_normal((1, tokens, heads, R.D))).astype(np.float16)
    got = _attend(ctx, k, v, 1, q, out_type)
    ref, smax, vmax = R.attention(q, k[None, None], v[None, None], [n], [tokens])
    bf16, many = out_type == TYPE_BF16, tokens * heads > 16
    tol = R.attention_tolerance(ref, smax, vmax, 2.0 ** -7 if bf16 else 2.0 ** -10, bf16 and many, bf16 and not many)
    assert np.all(np.abs(got - ref) <= tol), np.max(np.abs(got - ref) / tol)
