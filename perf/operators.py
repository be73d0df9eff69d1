"""The operators of a decoder layer with a sliding window, as cases that can be timed and compared:
attention with a window and first tokens that stay visible (prefill, training, single tokens over a
cache), rotary positions with several axes, and the root-mean-square norm with an 8-bit output.

``run`` computes a case in plain torch operations where ``own`` is false, and through the entry points
of ``inductor_x_b200.ops`` where it is true.  ``exact`` computes it in 64 bits from the definition.
"""
import math

import torch

#: set by whoever measures: the package's operators instead of their plain forms
own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
HEAD = 128        # head dimension of the attention
GROUP = 128       # values that share a scale, where the scales are not the rows'
EPS = 1e-6
LARGEST = 448.0   # of an 8-bit value of four exponent and three mantissa bits


def listed():
    return [
        # prefill of a long prompt in one sequence, four query heads to a key head
        {"name": "attention_prefill", "kind": "attention", "dtype": "bf16", "b": 1, "heads": 32, "kv_heads": 8,
         "queries": 8192, "keys": 8192, "window": 1024, "sinks": 4, "ragged": False},
        # the next chunk of three prompts of different lengths, padded to the longest, behind what the cache has of each
        {"name": "attention_chunk_ragged", "kind": "attention", "dtype": "f16", "b": 3, "heads": 12, "kv_heads": 4,
         "queries": 500, "keys": 2100, "window": 600, "sinks": 5, "ragged": True},
        # one token of one sequence: what a user who waits for an answer sees
        {"name": "attention_decode_one", "kind": "attention", "dtype": "bf16", "b": 1, "heads": 32, "kv_heads": 8,
         "queries": 1, "keys": 8192, "window": 1024, "sinks": 4, "ragged": False},
        # one token of each of 64 sequences that are anywhere in their cache: a server's step
        {"name": "attention_decode_batch", "kind": "attention", "dtype": "bf16", "b": 64, "heads": 32, "kv_heads": 8,
         "queries": 1, "keys": 16384, "window": 4096, "sinks": 4, "ragged": True},
        # a training step over 2 x 4096 tokens: output and all gradients
        {"name": "attention_training", "kind": "attention_training", "dtype": "bf16", "b": 2, "heads": 32, "kv_heads": 8,
         "queries": 4096, "keys": 4096, "window": 1024, "sinks": 4, "ragged": False},
        # the same with a key head to each query head, on lengths that are no whole number of tiles
        {"name": "attention_training_odd", "kind": "attention_training", "dtype": "f16", "b": 1, "heads": 8, "kv_heads": 8,
         "queries": 1531, "keys": 1531, "window": 257, "sinks": 16, "ragged": False},
        # a server's step: one token of 16 sequences
        {"name": "rotary_decode", "kind": "rotary", "dtype": "bf16", "b": 16, "s": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "sections": "16,24,24", "pairing": "halves", "ladder": "shared", "far": 30000, "inverse": False, "storage": "bshd"},
        # a training step over video and text: three axes, forward and backward
        {"name": "rotary_training", "kind": "rotary", "dtype": "bf16", "b": 2, "s": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "sections": "16,24,24", "pairing": "halves", "ladder": "shared", "far": 100000, "inverse": True, "storage": "bshd"},
        # the patches of images, 37 x 37 each: two axes with frequencies of their own, heads of 80
        {"name": "rotary_image", "kind": "rotary", "dtype": "f16", "b": 3, "s": 1369, "heads": 16, "kv_heads": 16, "dim": 80,
         "sections": "20,20", "pairing": "neighbours", "ladder": "own", "far": 37, "inverse": False, "storage": "bhsd"},
        # one decoding step of 16 sequences
        {"name": "norm_decode", "kind": "norm", "dtype": "bf16", "rows": 16, "cols": 4096, "group": 0, "residual": True},
        # prefill of 16384 tokens, a scale for each 128 values as a blockwise product wants them
        {"name": "norm_prefill", "kind": "norm", "dtype": "bf16", "rows": 16384, "cols": 4096, "group": GROUP, "residual": True},
        # rows of odd length without a residual: no row but the first starts on a 16-byte boundary
        {"name": "norm_odd", "kind": "norm", "dtype": "f16", "rows": 5003, "cols": 1537, "group": GROUP, "residual": False},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm, odd ones among them."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _heads(rng, most):
    """(query heads, key heads): groups of one to eight, not always a power of two."""
    kv = rng.choice([n for n in (1, 2, 3, 4, 8, 16) if n <= most])
    return kv * rng.choice([n for n in (1, 1, 2, 3, 4, 5, 7, 8) if kv * n <= most]), kv


def draw(rng):
    kind = rng.choice(["prefill", "decode", "decode", "attention_training", "rotary", "rotary", "norm", "norm"])
    half = rng.choice(["f16", "bf16"])
    anyt = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("prefill", "attention_training"):
        most = 1 << 30 if kind == "prefill" else 1 << 29  # scores of the plain form
        heads, kv = _heads(rng, 32)
        b = rng.choice([1, 1, 2, 3])
        queries = _log(rng, 17, 6000)
        queries = min(queries, int(math.sqrt(most / (b * heads))))
        keys = queries if rng.random() < 0.5 else queries + _log(rng, 1, 2000)
        keys = max(queries, min(keys, most // (b * heads * queries)))
        return {"kind": "attention" if kind == "prefill" else kind, "dtype": half, "b": b, "heads": heads, "kv_heads": kv,
                "queries": queries, "keys": keys, "window": _log(rng, 16, 4096), "sinks": rng.choice([0, 1, 4, 7, 32, 64]),
                "ragged": rng.random() < 0.4}
    if kind == "decode":
        heads, kv = _heads(rng, 64)
        keys = _log(rng, 100, 32768)
        return {"kind": "attention", "dtype": half, "b": min(_log(rng, 1, 64), max(1, (1 << 22) // (keys * kv))), "heads": heads,
                "kv_heads": kv, "queries": rng.choice([1, 1, 1, 2, 3, 4]), "keys": keys, "window": _log(rng, 64, 4096),
                "sinks": rng.choice([0, 1, 4, 7, 32, 64]), "ragged": rng.random() < 0.6}
    if kind == "rotary":
        sections, dim = rng.choice([("64", 128), ("16,24,24", 128), ("32,32", 128), ("22,21,21", 128), ("20,20", 80),
                                    ("8,12,12", 64), ("16,16", 96), ("8,28,28", 128), ("10,11,11", 64), ("16,16,16,16", 128)])
        heads, kv = _heads(rng, 32)
        b = rng.choice([1, 1, 2, 4, 16])
        s = _log(rng, 1, max(1, 400000 // (b * heads)))
        return {"kind": kind, "dtype": anyt, "b": b, "s": s, "heads": heads, "kv_heads": kv, "dim": dim, "sections": sections,
                "pairing": rng.choice(["halves", "halves", "neighbours"]), "ladder": rng.choice(["shared", "shared", "own"]),
                "far": _log(rng, 30, 1000000), "inverse": rng.random() < 0.4, "storage": rng.choice(["bshd", "bshd", "bhsd"])}
    cols = rng.choice([_log(rng, 100, 16384), 64 * _log(rng, 2, 256)])
    return {"kind": "norm", "dtype": anyt, "rows": _log(rng, 1, (1 << 25) // cols), "cols": cols, "group": rng.choice([0, GROUP]),
            "residual": rng.random() < 0.7}


# ---- inputs --------------------------------------------------------------------------------------
def _lengths(case):
    """(lengths of the queries, lengths of the keys) of each sequence: the first has all of them, another nothing at all."""
    b, queries, keys = case["b"], case["queries"], case["keys"]
    if not case["ragged"]:
        return [queries] * b, [keys] * b
    kv = [keys if i == 0 else 0 if i == 2 else keys - 1 - (i * 7919) % keys for i in range(b)]
    return [queries] * b if queries <= 4 else [queries - (i * 31) % queries for i in range(b)], kv


def _sections(case):
    return [int(n) for n in case["sections"].split(",")]


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    new = lambda *shape: torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)  # noqa: E731
    state = {"case": case}
    if case["kind"] in ("attention", "attention_training"):
        b, h, kv, s, n = (case[k] for k in ("b", "heads", "kv_heads", "queries", "keys"))
        # queries as a projection leaves them, [B, S, H, D] in memory; keys and values as a cache (or, in training, a
        # projection) holds them
        state["q"] = new(b, s, h, HEAD).transpose(1, 2)
        if case["kind"] == "attention":
            state["k"], state["v"] = (torch.randn(b, kv, n, HEAD, generator=gen, device=dev, dtype=dtype) for _ in range(2))
        else:
            state["k"], state["v"] = new(b, n, kv, HEAD).transpose(1, 2), new(b, n, kv, HEAD).transpose(1, 2)
            state["dout"] = new(b, s, h, HEAD).transpose(1, 2)
        if case["ragged"]:
            ql, kl = _lengths(case)
            state["kv_lengths"] = torch.tensor(kl, dtype=torch.int32, device=dev)
            state["q_lengths"] = torch.tensor(ql, dtype=torch.int32, device=dev) if s > 4 else None
        else:
            state["kv_lengths"] = state["q_lengths"] = None
    elif case["kind"] == "rotary":
        b, s, d = case["b"], case["s"], case["dim"]
        for name, h in (("q", case["heads"]), ("k", case["kv_heads"])):
            state[name] = new(b, s, h, d).transpose(1, 2) if case["storage"] == "bshd" else new(b, h, s, d)
            if case["inverse"]:
                state["d" + name] = new(b, s, h, d).transpose(1, 2) if case["storage"] == "bshd" else new(b, h, s, d)
        # positions along each axis: the first far out (a long text), the others within a frame
        axes = len(_sections(case))
        state["positions"] = torch.stack([
            torch.randint(0, case["far"] if a == 0 else min(case["far"], 128), (b, s), generator=gen, device=dev)
            for a in range(axes)])
    else:
        rows, cols = case["rows"], case["cols"]
        state["x"] = new(rows, cols)
        state["residual"] = new(rows, cols) if case["residual"] else None
        state["w"] = (1 + 0.1 * torch.randn(cols, generator=gen, device=dev)).to(dtype)
    return state


# ---- plain forms -----------------------------------------------------------------------------------
def _visible(case, ql, kl, places, dev):
    """[B, 1, 1, queries, n]: which of the keys at ``places`` [B or 1, n] each query sees."""
    i = torch.arange(case["queries"], device=dev)
    at = (kl - ql)[:, None] + i                                                    # positions of the queries
    p, j = at[:, :, None], places[:, None, :]
    seen = (j <= p) & ((j > p - case["window"]) | (j < case["sinks"])) & (j >= 0) & (j < kl[:, None, None])
    return (seen & (i < ql[:, None])[:, :, None])[:, None, None]


def _plain_attention(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    b, h, n_q, _ = q.shape
    kv, n = k.shape[1], k.shape[2]
    dev = q.device
    ql = s["q_lengths"].long() if s["q_lengths"] is not None else torch.full((b,), n_q, device=dev)
    kl = s["kv_lengths"].long() if s["kv_lengths"] is not None else torch.full((b,), n, device=dev)
    reach = case["window"] + n_q - 1
    places = torch.arange(n, device=dev)[None]
    if case["kind"] == "attention" and 2 * (reach + case["sinks"]) < n:
        # few keys of a long cache: the first ones and the window's are picked, each once
        begin = (kl - reach).clamp(min=case["sinks"])
        places = torch.cat([torch.arange(case["sinks"], device=dev).expand(b, -1),
                            begin[:, None] + torch.arange(reach, device=dev)], dim=1)
        pick = places.clamp(max=n - 1)
        rows = torch.arange(b, device=dev)[:, None]
        k, v = k[rows, :, pick].transpose(1, 2), v[rows, :, pick].transpose(1, 2)
    q, k, v = q.float().reshape(b, kv, h // kv, n_q, HEAD), k.float()[:, :, None], v.float()[:, :, None]
    scale = HEAD ** -0.5
    scores = (q @ k.transpose(-1, -2)) * scale
    scores = scores.masked_fill(~_visible(case, ql, kl, places, dev), -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).reshape(b, h, n_q)
    p = p / torch.where(total > 0, total, 1.0)
    out = p @ v
    dtype = s["q"].dtype
    if case["kind"] == "attention":
        return out.reshape(b, h, n_q, HEAD).to(dtype), lse
    go = s["dout"].float().reshape(b, kv, h // kv, n_q, HEAD)
    ds = p * (go @ v.transpose(-1, -2) - (go * out).sum(-1, keepdim=True)) * scale
    dq = ds @ k
    # a key head's gradient is the sum over the query heads that share it
    flat = lambda t: t.reshape(b, kv, -1, t.shape[-1])  # noqa: E731
    dk, dv = flat(ds).transpose(-1, -2) @ flat(q), flat(p).transpose(-1, -2) @ flat(go)
    return (out.reshape(b, h, n_q, HEAD).to(dtype), lse, dq.reshape(b, h, n_q, HEAD).to(dtype), dk.to(dtype), dv.to(dtype))


def _plain_rotary(s):
    case = s["case"]
    sections, d, dev = _sections(case), case["dim"], s["q"].device
    pairs = sum(sections)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=dev)
    i = torch.arange(pairs, device=dev, dtype=torch.float64)
    if case["ladder"] == "own":
        i = torch.tensor([j / n for n in sections for j in range(n)], device=dev, dtype=torch.float64)
    else:
        i = i / pairs
    # the angle of a far position keeps nothing of its fraction in 32 bits
    angle = s["positions"][axis].double().permute(1, 2, 0)[:, None] * 10000.0 ** -i
    cos, sin = angle.cos().float(), angle.sin().float()

    def turn(x, sin):
        r, rest = x[..., :2 * pairs].float(), x[..., 2 * pairs:]
        if case["pairing"] == "halves":
            a, c = r[..., :pairs], r[..., pairs:]
            y = torch.cat([a * cos - c * sin, a * sin + c * cos], -1)
        else:
            a, c = r[..., 0::2], r[..., 1::2]
            y = torch.stack([a * cos - c * sin, a * sin + c * cos], -1).flatten(-2)
        return torch.cat([y.to(x.dtype), rest], -1)

    out = turn(s["q"], sin), turn(s["k"], sin)
    return out + (turn(s["dq"], -sin), turn(s["dk"], -sin)) if case["inverse"] else out


def _plain_norm(s):
    x, group = s["x"], s["case"]["group"]
    h = x if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype)
    f = h.float()
    y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * s["w"].float()
    rows, cols = y.shape
    width = group or cols
    padded = torch.nn.functional.pad(y, (0, -cols % width)).view(rows, -1, width)
    scales = padded.abs().amax(-1) / LARGEST
    scaled = padded / torch.where(scales > 0, scales, 1.0)[..., None]
    q = scaled.clamp(-LARGEST, LARGEST).view(rows, -1)[:, :cols].to(torch.float8_e4m3fn)
    scales = scales if group else scales[:, 0]
    return (q, scales, h) if s["residual"] is not None else (q, scales)


def run(state):
    case = state["case"]
    if own:
        from inductor_x_b200 import ops

        if case["kind"] in ("attention", "attention_training"):
            mask = {"window": case["window"], "sinks": case["sinks"], "q_lengths": state["q_lengths"],
                    "kv_lengths": state["kv_lengths"]}
            q, k, v = state["q"], state["k"], state["v"]
            out, lse = ops.window_attention(q, k, v, HEAD ** -0.5, return_lse=True, **mask)
            if case["kind"] == "attention":
                return out, lse
            return (out, lse) + tuple(ops.window_attention_backward(q, k, v, out, lse, state["dout"], HEAD ** -0.5, **mask))
        if case["kind"] == "rotary":
            turn = {"sections": _sections(case), "base": 10000.0, "pairing": case["pairing"], "ladder": case["ladder"]}
            out = tuple(ops.axial_rotary(state["q"], state["k"], state["positions"], **turn))
            if not case["inverse"]:
                return out
            return out + tuple(ops.axial_rotary_backward(state["dq"], state["dk"], state["positions"], **turn))
        return ops.rmsnorm_quantised(state["x"], state["w"], EPS, residual=state["residual"],
                                     return_residual=state["residual"] is not None, group=case["group"])
    if case["kind"] in ("attention", "attention_training"):
        return _plain_attention(state)
    return _plain_rotary(state) if case["kind"] == "rotary" else _plain_norm(state)


# ---- the definition in 64 bits -----------------------------------------------------------------------
def _exact_attention(case, s):
    q, k, v = s["q"], s["k"], s["v"]
    share, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(HEAD)
    training = case["kind"] == "attention_training"
    new = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)  # noqa: E731
    out, dq, dk, dv = new(q), new(q), new(k), new(v)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    for b, (n_q, n_k) in enumerate(zip(*_lengths(case))):
        first = n_k - n_q                        # the position of the first query
        skip = max(0, -first)                    # queries before the first key see nothing
        if n_q - skip <= 0 or n_k <= 0:
            continue
        at = torch.arange(first + skip, n_k, device=q.device)[:, None]
        low = max(0, first + skip - case["window"] + 1)
        keys = torch.cat([torch.arange(min(case["sinks"], low), device=q.device), torch.arange(low, n_k, device=q.device)])
        hidden = (keys > at) | ((at - keys >= case["window"]) & (keys >= case["sinks"]))
        for g in range(case["kv_heads"]):
            kd, vd = k[b, g, keys].double(), v[b, g, keys].double()
            for h in range(g * share, (g + 1) * share):
                qd = q[b, h, skip:n_q].double()
                z = torch.where(hidden, -math.inf, scale * (qd @ kd.T))
                l = torch.logsumexp(z, 1)
                p = torch.exp(z - l[:, None])
                o = p @ vd
                out[b, h, skip:n_q], lse[b, h, skip:n_q] = o, l
                if training:
                    g_o = s["dout"][b, h, skip:n_q].double()
                    dz = p * (g_o @ vd.T - torch.sum(g_o * o, 1, keepdim=True))
                    dq[b, h, skip:n_q] = scale * (dz @ kd)
                    dk[b, g, keys] += scale * (dz.T @ qd)
                    dv[b, g, keys] += p.T @ g_o
    return (out, lse, dq, dk, dv) if training else (out, lse)


def _exact_rotary(case, s):
    sections, pairs = _sections(case), sum(_sections(case))

    def turn(x, sign):
        y = x.double()
        first = 0
        for a, n in enumerate(sections):
            for j in range(n):
                i = first + j
                power = j / n if case["ladder"] == "own" else i / pairs
                angle = sign * s["positions"][a].double() * math.pow(10000.0, -power)
                c, sn = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
                lo, hi = (i, i + pairs) if case["pairing"] == "halves" else (2 * i, 2 * i + 1)
                u, w = x[..., lo].double(), x[..., hi].double()
                y[..., lo], y[..., hi] = u * c - w * sn, w * c + u * sn
            first += n
        return y

    out = turn(s["q"], 1), turn(s["k"], 1)
    return out + (turn(s["dq"], -1), turn(s["dk"], -1)) if case["inverse"] else out


def _exact_norm(case, s):
    total = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
    h = total.to(s["x"].dtype).double()          # the row that is normalised is the rounded one
    y = h / torch.sqrt(torch.mean(h ** 2, 1, keepdim=True) + EPS) * s["w"].double()
    parts = torch.split(y, case["group"] or y.shape[1], dim=1)
    scales = [p.abs().max(1).values / LARGEST for p in parts]
    q = torch.cat([p / torch.where(c == 0, 1.0, c)[:, None] for p, c in zip(parts, scales)], 1)
    scales = torch.stack(scales, 1) if case["group"] else scales[0]
    return (q, scales, total) if s["residual"] is not None else (q, scales)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("attention", "attention_training"):
        return _exact_attention(case, state)
    return _exact_rotary(case, state) if case["kind"] == "rotary" else _exact_norm(case, state)


# ---- what a case cannot do without ---------------------------------------------------------------------
def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "norm":
        n = case["rows"] * case["cols"]
        scales = case["rows"] * (-(-case["cols"] // case["group"]) if case["group"] else 1)
        return {"bytes": n * (size * (3 if case["residual"] else 1) + 1) + case["cols"] * size + 4 * scales,
                "flops": n * (6 if case["residual"] else 5)}
    if case["kind"] == "rotary":
        tokens = case["b"] * case["s"]
        n = tokens * (case["heads"] + case["kv_heads"]) * case["dim"] * (2 if case["inverse"] else 1)
        return {"bytes": 2 * n * size + 8 * tokens * len(_sections(case)), "flops": 3 * n}
    pairs = keys = rows = 0
    for n_q, n_k in zip(*_lengths(case)):
        at = torch.arange(max(0, n_k - n_q), n_k, dtype=torch.int64) if n_k else torch.zeros(0, dtype=torch.int64)
        pairs += int((at + 1).clamp(max=case["window"]).sum() + (at + 1 - case["window"]).clamp(min=0, max=case["sinks"]).sum())
        low = max(0, int(at[0]) - case["window"] + 1) if len(at) else 0
        keys += (n_k - low) + min(case["sinks"], low)
        rows += len(at)
    training = case["kind"] == "attention_training"
    out_rows = case["b"] * case["queries"]
    moved = case["heads"] * HEAD * (rows + out_rows) + 2 * case["kv_heads"] * HEAD * keys
    if training:  # dout in, dq out, dk and dv out
        moved += case["heads"] * HEAD * (rows + out_rows) + 2 * case["kv_heads"] * HEAD * case["b"] * case["keys"]
    return {"bytes": size * moved + 4 * case["heads"] * out_rows,
            "flops": case["heads"] * pairs * HEAD * (14 if training else 4)}
