"""The operators of a 4-bit KV cache and of token sampling, as workloads.

    append   new key and value rows into a cache of 4-bit rows (Context.kv4_append),
             then those rows read back as the fp16 values the cache now holds
             (Context.kv4_read_f16)
    attend   grouped-query attention of one or many tokens over such a cache
             (Context.attn_kv4)
    sample   one token per row of logits by temperature, top-k, top-p and min-p
             from a given uniform number (Context.sample_f32)

``run`` computes each in its plain form (elementary torch operations), or, with
``own`` true, through metallm_b200.

A cache row of 80 bytes holds 128 values in four groups of 32: 64 bytes of codes
(element i in byte i / 2, the low nibble for even i), then four fp16 pairs (d, m).
Element i of group g stands for m_g + d_g c_i.  A row x is stored with, in 32-bit
arithmetic and per group, m = fp16(min x), d = fp16((max x - m) * (1/15)) and
c = round((x - m) (1 / d)) kept within 0 .. 15 (round half to even; 0 where d is 0);
x is first kept within -65408 .. 65408.  Caches are [batch][kv head][capacity][80].
"""
import math

import numpy as np
import torch

own = False

D = 128          # head dimension
GROUP = 32       # elements that share a scale
ROW = 80         # bytes of a cache row
LIMIT = 65408.0  # rows are kept within this, so that m + 15 d stays an fp16 value whatever d rounds to

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # a decode step's new row, straight out of the fused fp32 QKV projection
        {"name": "append, one token", "op": "append", "batch": 1, "tokens": 1, "n_heads": 32, "n_kv": 8,
         "capacity": 8192, "type": "f32", "fused": True, "ragged": False},
        # a prompt chunk of the runner, likewise
        {"name": "append, chunk of 1024", "op": "append", "batch": 1, "tokens": 1024, "n_heads": 32, "n_kv": 8,
         "capacity": 8192, "type": "f32", "fused": True, "ragged": False},
        # prompts of unequal length, padded to the longest, as fp16 rows
        {"name": "append, 16 ragged prompts", "op": "append", "batch": 16, "tokens": 509, "n_heads": 32, "n_kv": 8,
         "capacity": 2048, "type": "f16", "fused": False, "ragged": True},
        # one conversation, one new token, the cache of a usual chat
        {"name": "decode, 2048 rows", "op": "attend", "batch": 1, "tokens": 1, "n_heads": 32, "n_kv": 8,
         "length": 2048, "capacity": 8192, "out": "f16", "ragged": False},
        # one long document, one new token
        {"name": "decode, 131071 rows", "op": "attend", "batch": 1, "tokens": 1, "n_heads": 32, "n_kv": 8,
         "length": 131071, "capacity": 131072, "out": "f16", "ragged": False},
        # a full serving batch (64 query heads), outputs for the bf16 linears
        {"name": "decode, 64 sequences", "op": "attend", "batch": 64, "tokens": 1, "n_heads": 64, "n_kv": 8,
         "length": 8192, "capacity": 8192, "out": "bf16", "ragged": False},
        # sequences of unequal length, one of them empty
        {"name": "decode, 24 ragged", "op": "attend", "batch": 24, "tokens": 1, "n_heads": 32, "n_kv": 8,
         "length": 16000, "capacity": 16384, "out": "f16", "ragged": True},
        # four drafted tokens of each sequence checked at once
        {"name": "verify, 8 x 4 tokens", "op": "attend", "batch": 8, "tokens": 4, "n_heads": 32, "n_kv": 8,
         "length": 4099, "capacity": 8192, "out": "f16", "ragged": False},
        # the last chunk of a prompt behind the chunks already in the cache
        {"name": "prompt, 1024 at 8192", "op": "attend", "batch": 1, "tokens": 1024, "n_heads": 32, "n_kv": 8,
         "length": 8192, "capacity": 8192, "out": "bf16", "ragged": False},
        # padded chunks of several prompts, every head with keys of its own
        {"name": "prompt, 5 ragged", "op": "attend", "batch": 5, "tokens": 333, "n_heads": 16, "n_kv": 16,
         "length": 2500, "capacity": 4096, "out": "bf16", "ragged": True},
        # one conversation's next token with the usual chat settings
        {"name": "sample, one row", "op": "sample", "rows": 1, "n": 128256, "temperature": 0.8, "top_k": 40,
         "top_p": 0.95, "min_p": 0.05, "mixed": False},
        # a serving batch, each row with settings of its own
        {"name": "sample, 64 rows", "op": "sample", "rows": 64, "n": 128256, "temperature": 1.0, "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "mixed": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "sample"])
    if op == "append":
        # at most 65536 rows of keys, and as many of values, spread over 1 to 32 sequences
        n_kv = rng.choice([1, 2, 4, 8, 8, 8, 10, 16])
        batch = _log_int(rng, 1, 32)
        tokens = max(1, min(_log_int(rng, 1, 2048), 65536 // (n_kv * batch)))
        return {"op": op, "batch": batch, "tokens": tokens, "n_heads": n_kv * rng.choice([1, 2, 4, 8]), "n_kv": n_kv,
                "capacity": tokens + rng.randint(0, 2000), "type": rng.choice(["f32", "f32", "f16", "bf16"]),
                "fused": rng.random() < 0.5, "ragged": batch > 1 and rng.random() < 0.5}
    if op == "attend":
        n_heads, n_kv = rng.choice([(32, 8), (32, 8), (64, 8), (8, 8), (16, 8), (28, 4), (32, 2), (40, 8), (4, 1)])
        kind = rng.choice(["decode", "decode", "verify", "prompt"])
        if kind == "decode":
            # the cache read is at most the largest listed one's
            batch = _log_int(rng, 1, 64)
            tokens, length = 1, min(_log_int(rng, 1, 131072), 64 * 8 * 8192 // (batch * n_kv))
        elif kind == "verify":
            batch, tokens = _log_int(rng, 1, 16), rng.randint(2, 16)
            length = tokens + _log_int(rng, 1, 16384)
        else:
            # at most 2^35 products of q and k
            batch, tokens = _log_int(rng, 1, 8), _log_int(rng, 17, 1024)
            length = tokens + min(_log_int(rng, 1, 16384), max(1, (1 << 28) // (batch * tokens * n_heads)))
        return {"op": op, "batch": batch, "tokens": tokens, "n_heads": n_heads, "n_kv": n_kv, "length": length,
                "capacity": length + rng.randint(0, 300),
                "out": "bf16" if kind == "prompt" or batch > 1 and rng.random() < 0.5 else "f16",
                "ragged": batch > 1 and rng.random() < 0.5}
    rows = _log_int(rng, 1, 64)
    return {"op": op, "rows": rows, "n": _log_int(rng, 500, 128256), "temperature": rng.choice([0.3, 0.7, 1.0, 1.3]),
            "top_k": rng.choice([0, 0, 1, 20, 50, 1000]), "top_p": rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]),
            "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]), "mixed": rng.random() < 0.3}


def _counts(case):
    """Tokens of each sequence: all of them, or between one and all, the last sequence none."""
    B, T = case["batch"], case["tokens"]
    if not case["ragged"] or T == 1:
        return [T] * B
    return [1 + (T - 1) * ((b * 7) % B + 1) // B for b in range(B - 1)] + [0]


def _lengths(case):
    """Cached rows of each sequence, its new ones among them; spread where ragged, the second sequence empty."""
    B, L, counts = case["batch"], case["length"], _counts(case)
    if not case["ragged"]:
        return [L] * B
    lens = [max(c, L * ((b * 5) % B + 1) // B) for b, c in enumerate(counts)]
    if B > 1 and case["tokens"] == 1:
        lens[1] = 0
    return lens


def work(case):
    if case["op"] == "append":
        n = sum(_counts(case)) * case["n_kv"] * 2           # rows, K and V
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": n * (D * size + ROW) + n * (ROW + 2 * D), "flops": 6 * n * D}
    if case["op"] == "attend":
        pairs = rows = 0
        for n, c in zip(_lengths(case), _counts(case)):
            rows += n
            pairs += max(0, n) if case["tokens"] == 1 else c * (n - c) + c * (c + 1) // 2
        q = sum(_counts(case)) * case["n_heads"] * D
        return {"bytes": rows * case["n_kv"] * 2 * ROW + 4 * q, "flops": 4 * pairs * case["n_heads"] * D}
    return {"bytes": case["rows"] * (4 * case["n"] + 28), "flops": 10 * case["rows"] * case["n"]}


# ---- inputs -----------------------------------------------------------------

def _quantize(x):
    """Rows [..., 128] to cache rows [..., 80]."""
    x = x.float().clamp(-LIMIT, LIMIT).unflatten(-1, (D // GROUP, GROUP))
    m = x.amin(-1, keepdim=True).half()
    d = ((x.amax(-1, keepdim=True) - m.float()) * (1.0 / 15.0)).half()
    inv = torch.where(d > 0, 1.0 / d.float(), torch.zeros_like(d, dtype=torch.float32))
    c = torch.round((x - m.float()) * inv).clamp(0, 15).to(torch.uint8).flatten(-2)
    codes = c[..., 0::2] | (c[..., 1::2] << 4)
    scales = torch.cat([d, m], -1).flatten(-2).contiguous().view(torch.uint8)
    return torch.cat([codes, scales], -1)


def _values(rows):
    """Cache rows [..., 80] to the fp32 values [..., 128] they stand for."""
    codes = rows[..., :D // 2]
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (D // GROUP, GROUP))
    s = rows[..., D // 2:].contiguous().view(torch.float16).unflatten(-1, (D // GROUP, 2)).float()
    return (c * s[..., :1] + s[..., 1:]).flatten(-2)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "append":
        B, T, H = case["batch"], case["tokens"], case["n_kv"]
        width = (case["n_heads"] + 2 * H) * D if case["fused"] else H * D
        src = [torch.randn(B, T, width, generator=g, device="cuda").to(_TYPES[case["type"]])
               for _ in range(1 if case["fused"] else 2)]
        for s in src:                       # some channels of keys are far larger than the others
            s[..., 5::61] *= 8
        k0 = case["n_heads"] * D if case["fused"] else 0
        counts = _counts(case)
        pos = [(b * 211) % (case["capacity"] - T + 1) for b in range(B)]
        return {"case": case, "src": src, "k": src[0][..., k0:k0 + H * D],
                "v": src[-1][..., k0 + H * D:k0 + 2 * H * D] if case["fused"] else src[1],
                "stride": width, "pos": _ints(pos), "counts": _ints(counts) if case["ragged"] else None,
                "cache": [torch.zeros(B, H, case["capacity"], ROW, dtype=torch.uint8, device="cuda") for _ in "kv"],
                "out": [torch.zeros(B, T, H, D, dtype=torch.float16, device="cuda") for _ in "kv"]}
    if case["op"] == "attend":
        B, T, NH, H, S = (case[k] for k in ("batch", "tokens", "n_heads", "n_kv", "capacity"))
        q = 1.5 * torch.randn(B, T, NH, D, generator=g, device="cuda")
        cache = []
        for _ in "kv":
            rows = torch.empty(B, H, S, ROW, dtype=torch.uint8, device="cuda")
            for b in range(B):
                x = torch.randn(H, S, D, generator=g, device="cuda")
                x[..., 5::61] *= 4
                rows[b] = _quantize(x)
            cache.append(rows)
        return {"case": case, "q": q.half(), "cache": cache, "lengths": _ints(_lengths(case)),
                "counts": _ints(_counts(case)) if case["ragged"] and T > 1 else None,
                "out": torch.zeros(B, T, NH, D, dtype=_TYPES[case["out"]], device="cuda")}
    R, n = case["rows"], case["n"]
    # most tokens unlikely, a few that compete
    logits = 2.2 * torch.randn(R, n, generator=g, device="cuda") - 3.0
    logits.scatter_add_(1, torch.randint(n, (R, 40), generator=g, device="cuda"),
                        12.0 * torch.rand(R, 40, generator=g, device="cuda"))
    p = [[case["temperature"], case["top_k"], case["top_p"], case["min_p"]] for _ in range(R)]
    if case["mixed"]:
        other = [[0.0, 0, 1.0, 0.0], [0.7, 50, 0.95, 0.0], [1.0, 0, 1.0, 0.05], [1.0, 0, 1.0, 0.0]]
        p = [p[r] if r % 5 == 0 else other[r % 5 - 1] for r in range(R)]
    params = torch.tensor(p, dtype=torch.float32)
    params[:, 1] = torch.tensor([int(r[1]) for r in p], dtype=torch.int32).view(torch.float32)
    return {"case": case, "logits": logits, "params": params.cuda(), "u": torch.rand(R, generator=g, device="cuda"),
            "token": torch.zeros(R, dtype=torch.int32, device="cuda"),
            "prob": torch.zeros(R, dtype=torch.float32, device="cuda")}


# ---- the plain form ---------------------------------------------------------

def _append(s):
    c = s["case"]
    B, T, H = c["batch"], c["tokens"], c["n_kv"]
    t = torch.arange(T, device="cuda")
    slot = (s["pos"].long()[:, None] + t)[:, None, :, None].expand(B, H, T, ROW)
    live = (t < s["counts"].long()[:, None])[:, None, :, None] if s["counts"] is not None else None
    for x, cache, out in zip((s["k"], s["v"]), s["cache"], s["out"]):
        new = _quantize(x.unflatten(-1, (H, D))).transpose(1, 2)
        if live is not None:
            new = torch.where(live, new, cache.gather(2, slot))
        cache.scatter_(2, slot, new)
        back = _values(cache.gather(2, slot)).half()
        if live is not None:
            back = torch.where(live, back, out.transpose(1, 2))
        out.copy_(back.transpose(1, 2))
    return s["out"]


def _attend(s):
    c = s["case"]
    B, T, NH, H, L = c["batch"], c["tokens"], c["n_heads"], c["n_kv"], c["length"]
    G = NH // H
    K, V = (_values(x[:, :, :L]) for x in s["cache"])
    q = s["q"].float().view(B, T, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * T, D)
    x = (q @ K.transpose(-1, -2)).mul_(1.0 / math.sqrt(D)).view(B, H, G, T, L)
    t = torch.arange(T, device="cuda")
    n = s["lengths"].long()
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(n, T)
    seen = (n - counts + 1)[:, None] + t                    # rows that token t attends to
    hidden = torch.arange(L, device="cuda") >= seen[..., None]
    x.masked_fill_(hidden[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = (x.view(B, H, G * T, L) @ V).view(B, H, G, T, D) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, NH, D).to(s["out"].dtype)
    if s["counts"] is not None:
        o = torch.where((t < counts[:, None])[..., None, None], o, s["out"])
    s["out"].copy_(o)
    return s["out"]


def _sample(s):
    x = s["logits"].double()
    T, k, top_p, min_p = s["params"].unbind(1)
    T, top_p, min_p = T.double()[:, None], top_p.double()[:, None], min_p.double()[:, None]
    k = k.contiguous().view(torch.int32)[:, None]
    R, n = x.shape
    k = torch.where((k <= 0) | (T <= 0), torch.where(T <= 0, 1, n), k)
    xs, order = x.sort(dim=1, descending=True, stable=True)
    w = torch.exp((xs - xs[:, :1]) / torch.where(T <= 0, torch.ones_like(T), T))
    rank = torch.arange(n, device="cuda")[None]
    w = torch.where(rank < k, w, torch.zeros_like(w))
    before = w.cumsum(1) - w
    keep = (rank == 0) | (before < top_p * w.sum(1, keepdim=True)) & (w >= min_p) & (w > 0)
    kept = torch.zeros_like(x).scatter_(1, order, torch.where(keep, w, torch.zeros_like(w)))
    at = kept.cumsum(1)
    total = at[:, -1:]
    token = (at <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    s["token"].copy_(token[:, 0])
    s["prob"].copy_((kept.gather(1, token) / total)[:, 0])
    return [s["token"], s["prob"]]


# ---- the framework's calls --------------------------------------------------

_contexts = {}  # of each device: the package, the context, the stream it is on


def _own_context(device):
    """The program's context of a device, on torch's current stream there (asked for as a raw
    handle: a Stream object takes 1 to 3 us to make)."""
    stream = torch._C._cuda_getCurrentRawStream(device)
    at = _contexts.get(device)
    if at is None:
        import metallm_b200
        at = _contexts[device] = [metallm_b200, metallm_b200.Context(device), None]
    if at[2] != stream:
        at[1].set_stream(stream or 1)  # 1: the default stream's handle
        at[2] = stream
    return at


def _own(s):
    c = s["case"]
    M, ctx, _ = _own_context((s["token"] if c["op"] == "sample" else s["cache"][0]).get_device())
    if c["op"] == "sample":
        ctx.sample_f32(s["logits"].data_ptr(), c["rows"], c["n"], c["n"], s["params"].data_ptr(), s["u"].data_ptr(),
                       s["token"].data_ptr(), s["prob"].data_ptr())
        return [s["token"], s["prob"]]
    cache = M.Kv4Cache(s["cache"][0].data_ptr(), s["cache"][1].data_ptr(), c["batch"], c["n_kv"], D, c["capacity"])
    counts = s["counts"].data_ptr() if s["counts"] is not None else None
    if c["op"] == "append":
        ctx.kv4_append(cache, s["k"].data_ptr(), s["v"].data_ptr(),
                       {"f32": M.TYPE_F32, "f16": M.TYPE_F16, "bf16": M.TYPE_BF16}[c["type"]], s["stride"],
                       c["tokens"], s["pos"].data_ptr(), counts)
        ctx.kv4_read_f16(cache, c["tokens"], s["pos"].data_ptr(), counts, s["out"][0].data_ptr(),
                         s["out"][1].data_ptr())
        return s["out"]
    ctx.attn_kv4(cache, s["q"].data_ptr(), c["n_heads"], c["tokens"], s["lengths"].data_ptr(), counts,
                 s["out"].data_ptr(), M.TYPE_F16 if c["out"] == "f16" else M.TYPE_BF16)
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"append": _append, "attend": _attend, "sample": _sample}[state["case"]["op"]](state)


# ---- in 64 bits, from the definitions ----------------------------------------

def _exact_rows(x):
    """What the cache holds for fp32 rows x [..., 128] (numpy), in 64 bits: the codes are chosen in the 32-bit
    arithmetic that the format prescribes."""
    x = np.clip(x.astype(np.float32), -LIMIT, LIMIT)
    out = np.empty(x.shape, np.float64)
    for g in range(0, D, GROUP):
        y = x[..., g:g + GROUP]
        lo, hi = y.min(-1), y.max(-1)
        m = lo.astype(np.float16).astype(np.float32)
        d = ((hi - m) * np.float32(1 / 15)).astype(np.float16).astype(np.float32)
        inv = np.divide(np.float32(1), d, out=np.zeros_like(d), where=d > 0)
        c = np.minimum(np.maximum(np.rint((y - m[..., None]) * inv[..., None]), 0), 15)
        out[..., g:g + GROUP] = m[..., None].astype(np.float64) + d[..., None].astype(np.float64) * c
    return out


def _exact_append(case, s):
    B, T, H = case["batch"], case["tokens"], case["n_kv"]
    outs = []
    for x in (s["k"], s["v"]):
        y = _exact_rows(x.float().cpu().numpy().reshape(B, T, H, D))
        for b, c in enumerate(_counts(case)):
            y[b, c:] = 0.0
        outs.append(y)
    return outs


def _exact_cache(rows):
    """fp64 values of cache rows [H, n, 80] by their bytes."""
    b = rows.to(torch.int64)
    i = torch.arange(D, device=rows.device)
    code = (b[..., i // 2] >> (4 * (i % 2))) & 15
    half = rows[..., 64:].contiguous().view(torch.float16).double()
    return half[..., 2 * (i // GROUP) + 1] + half[..., 2 * (i // GROUP)] * code


def _exact_attend(case, s):
    T, NH, H = case["tokens"], case["n_heads"], case["n_kv"]
    G = NH // H
    out = torch.zeros(case["batch"], T, NH, D, dtype=torch.float64, device="cuda")
    for b, (n, c) in enumerate(zip(_lengths(case), _counts(case))):
        if n == 0 or c == 0:
            continue
        for h in range(H):
            k, v = (_exact_cache(x[b, h, :n]) for x in s["cache"])
            q = s["q"][b, :c, h * G:(h + 1) * G].double()
            x = torch.einsum("tgd,nd->tgn", q, k) / math.sqrt(D)
            last = torch.arange(n - c, n, device="cuda")[:, None, None]
            x = torch.where(torch.arange(n, device="cuda") <= last, x, torch.full_like(x, -math.inf))
            out[b, :c, h * G:(h + 1) * G] = torch.einsum("tgn,nd->tgd", torch.softmax(x, -1), v)
    return out


def _exact_sample(case, s):
    x, u = s["logits"].cpu().numpy().astype(np.float64), s["u"].cpu().numpy().astype(np.float64)
    params = s["params"].cpu()
    ks = params[:, 1].contiguous().view(torch.int32).numpy()
    params = params.numpy().astype(np.float64)
    tokens, probs = np.zeros(len(x), np.int32), np.zeros(len(x))
    for r, row in enumerate(x):
        T, top_p, min_p = params[r, 0], params[r, 2], params[r, 3]
        if T <= 0:
            tokens[r], probs[r] = int(np.argmax(row)), 1.0
            continue
        order = np.argsort(-row, kind="stable")
        if ks[r] > 0:
            order = order[:ks[r]]
        w = np.exp((row[order] - row[order[0]]) / T)
        done = np.searchsorted(np.cumsum(w), top_p * math.fsum(w), side="left") + 1  # the first that reach top_p
        order, w = order[:done], w[:done]
        order, w = order[w >= min_p * w[0]], w[w >= min_p * w[0]]
        by_index = np.argsort(order)
        order, w = order[by_index], w[by_index]
        at = np.searchsorted(np.cumsum(w), u[r] * math.fsum(w), side="right")
        at = min(int(at), len(w) - 1)
        tokens[r], probs[r] = order[at], w[at] / math.fsum(w)
    return [tokens, probs]


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](case, s)
