"""The operators of a pre-norm layer served with 4-bit weights, as calls whose speed counts: residual + RMS norm (in the
storage type or in 8 bits), Dense layers on 4-bit weights with group scales, attention with a sliding window and sinks.

A case names one of them by `op`:

    "norm"       s = x + residual, out = gamma * s / sqrt(mean(s^2) + eps); bits 0: out in the storage type, 8: whole numbers
                 of -127..127 with one scale per row
    "dense"      out = x w^T + bias (, GELU) with w = code * scale, codes of 4 bits, one fp16 scale for `group` columns of a
                 row of w; x is "f32", "f16" or "i8" (8 bits with a scale per row, as "norm" writes them), out is `dtype`
    "attention"  query i of a sequence stands at p = first + i and sees key j if j < length, the mask keeps j,
                 j <= p + right and (j >= p - left or j < sinks); a bound of -1 is none. Heads share keys and values in
                 groups of heads / kv_heads. `kind` "self": whole padded sequences, queries and keys out of one packed
                 projection; "step": the last `queries` tokens of sequences whose keys lie in a cache of `keys` rows

Sizes are those of the two model configurations (hidden 768 and 1024, heads of 64) and generic ones.
"""
import math

import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16}


def _norm(name, dtype, rows, hidden, bits=0, residual=True):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "hidden": hidden, "bits": bits, "residual": residual}


def _dense(name, x, dtype, tokens, width, features, group, bias=True, gelu=False):
    return {"name": name, "op": "dense", "x": x, "dtype": dtype, "tokens": tokens, "width": width, "features": features,
            "group": group, "bias": bias, "gelu": gelu}


def _attention(name, kind, dtype, batch, queries, keys, heads, kv_heads, size, left, right, sinks, shortest=0.25, masked="no"):
    """shortest: the shortest sequence's share of `keys` (lengths are spread evenly up to all of it); masked: "no", "padding"
    (lengths are given as a mask, as the encoder's requests give them) or "holes" (one key of 16 is masked beside the lengths)"""
    return {"name": name, "op": "attention", "kind": kind, "dtype": dtype, "batch": batch, "queries": queries, "keys": keys,
            "heads": heads, "kv_heads": kv_heads, "size": size, "left": left, "right": right, "sinks": sinks,
            "shortest": shortest, "masked": masked}


def listed():
    return [
        # one token of a base-sized fp32 model between two layers: the shortest call there is, all of it latency
        _norm("norm f32 1x768", "f32", 1, 768),
        # the layer boundary of a large batch of the large model: 256 sequences of 128 tokens
        _norm("norm f16 32768x1024", "f16", 32768, 1024),
        # eight sequences a token each, on the way into a Dense layer that takes 8 bits
        _norm("norm i8 f16 8x4096", "f16", 8, 4096, bits=8),
        # a prompt of odd length in fp32, rows that are no whole number of wavefronts
        _norm("norm i8 f32 4099x1000", "f32", 4099, 1000, bits=8),
        # one token through the large model's intermediate layer: a matrix-vector product with its GELU
        _dense("dense f16 1x1024-4096", "f16", "f16", 1, 1024, 4096, 128, gelu=True),
        # a short query of the base model in fp32 through the packed projection, a token more than a whole tile
        _dense("dense f32 33x768-2304", "f32", "f32", 33, 768, 2304, 64),
        # a few sequences, small groups, features that end inside a tile
        _dense("dense f16 7x4096-4100", "f16", "f16", 7, 4096, 4100, 32, bias=False),
        # 16 sequences a token each through the widest layer: 134 MB of weights
        _dense("dense i8 16x8192-32768", "i8", "f16", 16, 8192, 32768, 128, bias=False),
        # long documents through the large model's heads, every token seeing 512 on either side and the first one
        _attention("attention f16 self 4x4096", "self", "f16", 4, 4096, 4096, 16, 16, 64, 512, 512, 1),
        # a prompt taken in pieces: 517 more tokens of three sequences in fp32, the 512 last keys and four sinks
        _attention("attention f32 piece 3x517", "step", "f32", 3, 517, 2000, 12, 12, 64, 511, 0, 4, shortest=0.5, masked="holes"),
        # 32 sequences a token each, window of 4096 out of a cache of 8192, four heads to a key head
        _attention("attention f16 step 32x1", "step", "f16", 32, 1, 8192, 16, 4, 128, 4095, 0, 4, shortest=0.1),
        # one long sequence a token at a time in a layer without a window: few rows, a long axis
        _attention("attention f16 step 1x131072", "step", "f16", 1, 1, 131072, 16, 2, 128, -1, 0, 0, shortest=1.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_size(c) for c in listed())
    while True:
        c = _drawn(rng)
        if _size(c) <= most:
            c.pop("name")
            return c


def _drawn(rng):
    op = rng.choice(("norm", "dense", "attention"))
    dtype = rng.choice(("f32", "f16"))
    if op == "norm":
        hidden = rng.choice((768, 1024, 2048, 4096, 8192, _log(rng, 48, 9000)))
        rows = _log(rng, 1, min(32768, (1 << 25) // hidden))
        c = _norm("", dtype, rows, hidden, rng.choice((0, 8)), rng.random() < 0.75)
    elif op == "dense":
        group = rng.choice((32, 64, 128))
        width = group * _log(rng, 1, 8192 // group)
        features = min(_log(rng, 16, 32768), (1 << 27) // width)
        c = _dense("", rng.choice((dtype, "i8")), dtype, _log(rng, 1, 64), width, features, group, rng.random() < 0.5,
                   rng.random() < 0.3)
    else:
        size, kv = rng.choice((32, 64, 128)), rng.choice((1, 2, 4, 8))
        heads = kv * rng.choice((1, 2, 4, 7))
        left = rng.choice((-1, _log(rng, 16, 4096)))
        sinks = rng.choice((0, 1, 4, 70))
        if rng.random() < 0.5:
            batch, keys = _log(rng, 1, 8), _log(rng, 33, 4096)
            batch = max(1, min(batch, 400_000_000 // (heads * keys * keys)))
            c = _attention("", "self", dtype, batch, keys, keys, heads, kv, size, left, rng.choice((0, left)), sinks, 0.25,
                           rng.choice(("no", "padding", "holes")))
        else:
            queries = rng.choice((1, 1, _log(rng, 2, 700)))
            keys = max(queries, _log(rng, 300, 60000 if queries == 1 else 8000))
            batch = max(1, min(_log(rng, 1, 48), 100_000_000 // (heads * queries * keys), 50_000_000 // (kv * keys * size)))
            c = _attention("", "step", dtype, batch, queries, keys, heads, kv, size, left, 0, sinks,
                           max(queries / keys, rng.choice((0.1, 0.6))), rng.choice(("no", "holes")))
    return c


# ---------------------------------------------------------------------------- inputs


def _lengths(case):
    """The lengths of a case's sequences, from the shortest to the longest (which of them has which goes by the seed)."""
    b, keys = case["batch"], case["keys"]
    short = max(1, case["queries"] if case["kind"] == "step" else 1, int(math.ceil(keys * case["shortest"])))
    return [keys if b == 1 else keys - (keys - short) * i // (b - 1) for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = dict(case)
    if case["op"] == "norm":
        t = TYPES[case["dtype"]]
        rows, hidden = case["rows"], case["hidden"]
        # a residual stream has some channels that stand far out
        loud = 1 + 15 * (torch.rand(hidden, generator=g, device="cuda") < 0.01)
        state["x"] = normal(rows, hidden).to(t)
        state["residual"] = (2 * normal(rows, hidden) * loud).to(t) if case["residual"] else None
        state["gamma"] = (1 + 0.1 * normal(hidden)).to(t)
    elif case["op"] == "dense":
        t = TYPES[case["dtype"]]
        tokens, width, features, group = case["tokens"], case["width"], case["features"], case["group"]
        x = normal(tokens, width)
        if case["x"] == "i8":
            top = x.abs().amax(1, keepdim=True)
            state["x"], state["x_scales"] = torch.round(x * (127 / top)).to(torch.int8), (top / 127).reshape(-1)
        else:
            state["x"] = x.to(TYPES[case["x"]])
        # weights of standard deviation 0.02 as a quantiser leaves them: the group's largest is code 7 or -7
        w = normal(features, width // group, group).mul_(0.02)
        state["scales"] = (w.abs().amax(2) / 7).half()
        codes = torch.round(w / state["scales"].float()[:, :, None]).clamp_(-8, 7).to(torch.int8).view(features, width)
        del w
        # two codes a byte, the even column in the low half
        state["codes"] = (codes[:, 0::2] & 15 | codes[:, 1::2] << 4).view(torch.uint8)
        state["bias"] = (0.1 * normal(features)).to(t) if case["bias"] else None
        if own:
            from cubert_amd import kernels
            state["weights"] = kernels.w4_pack(state["codes"], state["scales"], group)
    else:
        t = TYPES[case["dtype"]]
        batch, nq, nk, size = case["batch"], case["queries"], case["keys"], case["size"]
        heads, kv = case["heads"], case["kv_heads"]
        if case["kind"] == "self":
            packed = normal(batch * nq, heads + 2 * kv, size).to(t).view(batch, nq, heads + 2 * kv, size)
            state["q"], state["k"], state["v"] = packed[:, :, :heads], packed[:, :, heads:heads + kv], packed[:, :, heads + kv:]
        else:
            state["q"] = normal(batch, nq, heads, size).to(t)
            state["k"] = torch.empty(batch, nk, kv, size, device="cuda", dtype=t).normal_(generator=g)
            state["v"] = torch.empty(batch, nk, kv, size, device="cuda", dtype=t).normal_(generator=g)
        order = torch.randperm(batch, generator=g, device="cuda")
        lengths = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]
        state["first"] = lengths - nq if case["kind"] == "step" else None
        state["lengths"], state["mask"] = lengths, None
        if case["masked"] == "padding":
            state["mask"] = (torch.arange(nk, device="cuda") < lengths[:, None]).to(torch.int8)
            state["lengths"] = None
        elif case["masked"] == "holes":
            state["mask"] = (torch.rand(batch, nk, generator=g, device="cuda") >= 1 / 16).to(torch.int8)
    return state


# ---------------------------------------------------------------------------- one pass


def _gelu(x):
    return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))


def _run_norm(s):
    t, hidden = TYPES[s["dtype"]], s["hidden"]
    if own:
        from cubert_amd import kernels
        if not s["bits"]:
            return kernels.res_rms_norm(s["x"], s["residual"], s["gamma"], EPS)
        codes, scales, total = kernels.res_rms_norm_i8(s["x"], s["residual"], s["gamma"], EPS)
    else:
        x = s["x"].float()
        x = x + s["residual"].float() if s["residual"] is not None else x
        total = x.to(t) if s["residual"] is not None else None
        rstd = 1 / torch.sqrt((x * x).sum(1) / hidden + EPS)
        if not s["bits"]:
            return (s["gamma"].float() * (x * rstd[:, None])).to(t), total
        # the norm's factor is the same for a whole row and drops out of the codes
        x = s["gamma"].float() * x
        top = x.abs().amax(1)
        codes = torch.round(x * (torch.full_like(top, 127) / top)[:, None]).to(torch.int8)
        scales = top * rstd / 127
    # what the 8 bits stand for, as a consumer that takes no 8 bits would have it
    values = torch.empty(s["rows"], hidden, dtype=t, device="cuda")
    torch.mul(codes, scales[:, None], out=values)
    return values, scales, total


def _run_dense(s):
    if own:
        from cubert_amd import kernels
        if s["x"].dtype == torch.int8:
            return kernels.dense_w4_i8(s["x"], s["x_scales"], s["weights"], s["bias"], s["gelu"], TYPES[s["dtype"]])
        return kernels.dense_w4(s["x"], s["weights"], s["bias"], s["gelu"])
    features, width = s["features"], s["width"]
    codes = torch.stack((s["codes"] << 4, s["codes"]), 2).view(features, width).view(torch.int8) >> 4
    w = (codes.view(features, -1, s["group"]).float() * s["scales"].float()[:, :, None]).view(features, width)
    x = s["x"].float()
    x = x * s["x_scales"][:, None] if s["x"].dtype == torch.int8 else x
    y = x @ w.t()
    y = y + s["bias"].float() if s["bias"] is not None else y
    return (_gelu(y) if s["gelu"] else y).to(TYPES[s["dtype"]])


def _run_attention(s):
    q, k, v, size = s["q"], s["k"], s["v"], s["size"]
    if own:
        from cubert_amd import kernels
        return kernels.attention_window(q, k, v, s["left"], s["right"], s["sinks"], first=s["first"], lengths=s["lengths"],
                                        mask=s["mask"])
    share = s["heads"] // s["kv_heads"]
    b, nq, nk, kv = s["batch"], s["queries"], s["keys"], s["kv_heads"]
    p = torch.arange(nq, device="cuda") + (s["first"][:, None] if s["first"] is not None else torch.zeros(b, 1, device="cuda", dtype=torch.int64))
    p, j = p[:, :, None], torch.arange(nk, device="cuda")
    seen = (j >= p - s["left"]) | (j < s["sinks"]) if s["left"] >= 0 else torch.ones_like(p, dtype=torch.bool) | (j >= 0)
    if s["right"] >= 0:
        seen = seen & (j <= p + s["right"])
    if s["lengths"] is not None:
        seen = seen & (j < s["lengths"][:, None, None]) & (p < s["lengths"][:, None, None])
    if s["mask"] is not None:
        seen = seen & (s["mask"][:, None, :] != 0)
    # the heads that share keys are rows of one product
    rows = q.float().view(b, nq, kv, share, size).permute(0, 2, 3, 1, 4).reshape(b, kv, share * nq, size)
    scores = rows @ k.float().permute(0, 2, 3, 1) * (1 / math.sqrt(size))
    seen = seen[:, None, None].expand(b, 1, share, nq, nk).reshape(b, 1, share * nq, nk)
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(3, keepdim=True)
    e = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = e.sum(3, keepdim=True)
    out = (e @ v.float().permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    return out.view(b, kv, share, nq, size).permute(0, 3, 1, 2, 4).reshape(b, nq, s["heads"], size).to(q.dtype)


def run(state):
    if state["op"] == "norm":
        return _run_norm(state)
    if state["op"] == "dense":
        return _run_dense(state)
    return _run_attention(state)


# ---------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n, r = case["rows"] * case["hidden"], case["residual"]
        out = n + 4 * case["rows"] if case["bits"] else n * e
        return {"bytes": n * e * (3 if r else 1) + case["hidden"] * e + out, "flops": n * (6 if case["bits"] else 4)}
    if case["op"] == "dense":
        t, w, f = case["tokens"], case["width"], case["features"]
        x = t * w * {"f32": 4, "f16": 2, "i8": 1}[case["x"]] + (4 * t if case["x"] == "i8" else 0)
        return {"bytes": f * w // 2 + 2 * f * (w // case["group"]) + x + t * f * e + (f * e if case["bias"] else 0),
                "flops": 2 * t * f * w}
    pairs = reached = rows = 0
    nq, left, right = case["queries"], case["left"], case["right"]
    for n in _lengths(case):
        first = n - nq if case["kind"] == "step" else 0
        # padding given as a mask leaves its queries in place; given as lengths it leaves them nothing
        p = torch.arange(first, first + nq if case["masked"] == "padding" else min(first + nq, n), dtype=torch.int64)
        high = torch.clamp(p + right, max=n - 1) if right >= 0 else torch.full_like(p, n - 1)
        low = torch.clamp(p - left, min=0) if left >= 0 else torch.zeros_like(p)
        near = torch.clamp(high - low + 1, min=0)
        far = torch.clamp(torch.minimum(torch.clamp(low, max=case["sinks"]), high + 1), min=0)
        pairs += int((near + far).sum())
        rows += p.numel()
        begin, end = int(low.min()), int(high.max()) + 1
        reached += max(0, end - begin) + min(case["sinks"], begin, end)
    size, heads, kv = case["size"], case["heads"], case["kv_heads"]
    kept = 15 / 16 if case["masked"] == "holes" else 1
    mask = 0 if case["masked"] == "no" else case["batch"] * case["keys"]
    moved = rows * heads * size * e + case["batch"] * nq * heads * size * e + 2 * reached * kv * size * e + mask
    return {"bytes": moved, "flops": 4 * size * heads * pairs * kept}


# ---------------------------------------------------------------------------- the same in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        total = s["x"].double()
        if s["residual"] is not None:
            total = total + s["residual"].double()
        y = total * s["gamma"].double() * (total.pow(2).mean(1, keepdim=True) + EPS).rsqrt()
        kept = total if s["residual"] is not None else None
        if not case["bits"]:
            return y, kept
        scales = y.abs().amax(1) / 127
        # values next to a border between two codes may fall to either side of it, so the values have none in 64 bits
        return None, scales, kept
    if case["op"] == "dense":
        c = s["codes"].to(torch.int16)
        c = torch.cat(((c & 15)[..., None], (c >> 4)[..., None]), -1).reshape(case["features"], -1)
        c = torch.where(c > 7, c - 16, c)
        x = s["x"].double()
        if case["x"] == "i8":
            x = x * s["x_scales"].double().unsqueeze(1)
        out = torch.zeros(case["tokens"], case["features"], dtype=torch.float64, device="cuda")
        at, step = 0, max(1, (1 << 27) // case["width"])
        while at < case["features"]:
            part = c[at:at + step].double() * s["scales"][at:at + step].double().repeat_interleave(case["group"], 1)
            out[:, at:at + step] = torch.matmul(x, part.transpose(0, 1))
            at += step
        if s["bias"] is not None:
            out += s["bias"].double()
        return out * 0.5 * torch.erfc(-out / math.sqrt(2.0)) if case["gelu"] else out
    b, nq, nk = case["batch"], case["queries"], case["keys"]
    q, k, v, share = s["q"], s["k"], s["v"], case["heads"] // case["kv_heads"]
    out = torch.zeros(b, nq, case["heads"], case["size"], dtype=torch.float64, device="cuda")
    keys = torch.arange(nk, device="cuda").unsqueeze(0)
    for i in range(b):
        n = nk if s["lengths"] is None else int(s["lengths"][i])
        at = torch.arange(nq, device="cuda").unsqueeze(1) + (0 if s["first"] is None else int(s["first"][i]))
        hidden = (keys >= n) | (at >= n)
        if case["right"] >= 0:
            hidden = hidden | (keys - at > case["right"])
        if case["left"] >= 0:
            hidden = hidden | ((at - keys > case["left"]) & (keys >= case["sinks"]))
        if s["mask"] is not None:
            hidden = hidden | (s["mask"][i] == 0).unsqueeze(0)
        blind = hidden.all(1, keepdim=True)
        for h in range(case["heads"]):
            z = torch.matmul(q[i, :, h].double(), k[i, :, h // share].double().t().contiguous()) / math.sqrt(case["size"])
            z = z.masked_fill(hidden, -float("inf")).masked_fill(blind, 0.0)
            z = (z - torch.logsumexp(z, 1, keepdim=True)).exp()
            out[i, :, h] = torch.matmul(z, v[i, :, h // share].double()).masked_fill(blind, 0.0)
    return out
