"""Measured calls of the operators around a quantised or draft-extended KV cache.

Four kinds of case, each a step that a serving program makes:

  rotary   queries and keys of new tokens turned to their positions: both pair layouts, part of the head, plain and
           context-extended frequencies, one token per sequence or a whole prompt
  cache    new key / value rows written to an 8-bit cache and the same rows read back from it, or (rows that are
           there already) a long stretch of the cache read back
  decode   one query token per sequence over the 8-bit cache, ragged lengths
  tree     a tree of drafted tokens per sequence over a dense or an 8-bit cache: every token sees the committed rows
           and its own ancestors among the drafted rows at the end of the cache

With `own` false the same results come from elementary tensor operations in 32 bits (angles in 64).
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}
SMALLEST_SCALE = 2.0 ** -126          # rows whose scale would be below the normal numbers are held as zeros


def listed():
    return [
        # one new token for each of 8 sequences, far into their contexts: a launch, hardly any bytes
        {"name": "rotary-token", "op": "rotary", "type": "bf16", "batch": 8, "tokens": 1, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rotary_dim": 128, "interleaved": False, "theta": 500000.0, "factor": 1.0, "first": 130000},
        # two long prompts, half of each head rotated, neighbouring pairs, context extended eightfold
        {"name": "rotary-prompt", "op": "rotary", "type": "f16", "batch": 2, "tokens": 8192, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "rotary_dim": 64, "interleaved": True, "theta": 10000.0, "factor": 8.0, "first": 0},
        # an odd chunk of a prompt in 32 bits, a head that is no power of two
        {"name": "rotary-odd", "op": "rotary", "type": "f32", "batch": 3, "tokens": 777, "heads": 12, "kv_heads": 4,
         "head_dim": 80, "rotary_dim": 32, "interleaved": False, "theta": 10000.0, "factor": 1.0, "first": 4096},
        # the row that one decode step adds for each of 16 sequences
        {"name": "cache-token", "op": "cache", "write": True, "type": "bf16", "code": "int8", "batch": 16, "tokens": 1,
         "kv_heads": 8, "head_dim": 128, "capacity": 4096},
        # four prompts written at once
        {"name": "cache-prompt", "op": "cache", "write": True, "type": "f16", "code": "e4m3", "batch": 4, "tokens": 8192,
         "kv_heads": 8, "head_dim": 128, "capacity": 8200},
        # a long cache read back for a consumer that wants dense rows
        {"name": "cache-read", "op": "cache", "write": False, "type": "bf16", "code": "int8", "batch": 1, "tokens": 100003,
         "kv_heads": 8, "head_dim": 64, "capacity": 100352},
        # one short sequence: latency
        {"name": "decode-short", "op": "decode", "type": "bf16", "code": "int8", "batch": 1, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "kv_len": 777, "ragged": False},
        # a serving batch at mixed lengths
        {"name": "decode-batch", "op": "decode", "type": "bf16", "code": "int8", "batch": 16, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "kv_len": 16384, "ragged": True},
        # few very long contexts
        {"name": "decode-long", "op": "decode", "type": "f16", "code": "e4m3", "batch": 4, "heads": 64, "kv_heads": 8,
         "head_dim": 128, "kv_len": 131071, "ragged": False},
        # a small tree for one sequence: latency
        {"name": "tree-short", "op": "tree", "type": "bf16", "code": "dense", "batch": 1, "tokens": 6, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "kv_len": 1023, "ragged": False, "shared_tree": True},
        # a tree of 26 tokens for each sequence of a serving batch, over a 16-bit cache
        {"name": "tree-batch", "op": "tree", "type": "bf16", "code": "dense", "batch": 8, "tokens": 26, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "kv_len": 16384, "ragged": True, "shared_tree": False},
        # wide trees over the 8-bit cache: 512 query rows share every key, more arithmetic than bytes
        {"name": "tree-wide", "op": "tree", "type": "f16", "code": "int8", "batch": 4, "tokens": 64, "heads": 64,
         "kv_heads": 8, "head_dim": 128, "kv_len": 32768, "ragged": False, "shared_tree": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "cache", "decode", "decode", "tree", "tree"])
    kind = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8])
    if op == "rotary":
        head = rng.choice([64, 80, 96, 128, 256])
        batch = rng.choice([1, 2, 3, 5, 8, 16])
        most = 2 * 8192 * 40 * 128 // (batch * kv * (group + 1) * head * (2 if kind == "f32" else 1))
        return {"op": op, "type": kind, "batch": batch, "tokens": _log(rng, 1, max(1, min(16384, most))), "heads": kv * group,
                "kv_heads": kv, "head_dim": head, "rotary_dim": rng.choice([head, head // 2, 32]),
                "interleaved": rng.random() < 0.5, "theta": rng.choice([10000.0, 500000.0, 10000000.0]),
                "factor": rng.choice([1.0, 1.0, 4.0, 16.0]), "first": _log(rng, 1, 200000)}
    if op == "cache":
        head = rng.choice([64, 96, 128, 256])
        batch = rng.choice([1, 2, 3, 4, 16])
        tokens = _log(rng, 1, min(32768, 4 * 8192 * 8 * 128 // (batch * kv * head * (2 if kind == "f32" else 1))))
        return {"op": op, "write": rng.random() < 0.7, "type": kind, "code": rng.choice(["int8", "e4m3"]), "batch": batch,
                "tokens": tokens, "kv_heads": kv, "head_dim": head, "capacity": tokens + rng.randint(0, 100)}
    head = rng.choice([64, 128, 128])
    batch = rng.choice([1, 2, 3, 4, 8, 16])
    rows = 4 * 8 * 131071 * 128 // (batch * kv * head)
    if op == "decode":
        return {"op": op, "type": kind, "code": rng.choice(["int8", "e4m3"]), "batch": batch, "heads": kv * group,
                "kv_heads": kv, "head_dim": head, "kv_len": _log(rng, 1, min(131071, rows // (4 if kind == "f32" else 1))),
                "ragged": rng.random() < 0.5}
    tokens = _log(rng, 2, 64)
    code = rng.choice(["dense", "dense", "int8", "e4m3"])
    most = 4 * 64 * 64 * 32768 * 128 // (batch * kv * group * tokens * head * (16 if kind == "f32" else 1))
    return {"op": op, "type": kind, "code": code, "batch": batch, "tokens": tokens, "heads": kv * group, "kv_heads": kv,
            "head_dim": head, "kv_len": _log(rng, tokens, max(tokens, min(32768, most))), "ragged": rng.random() < 0.5,
            "shared_tree": rng.random() < 0.5}


# ---- inputs -----------------------------------------------------------------------------------------------------
def _lengths(case):
    """The cache length of each sequence, by the case alone: between half of kv_len and all of it when ragged."""
    b, L, t = case["batch"], case["kv_len"], case.get("tokens", 1)
    if not case["ragged"]:
        return [L] * b
    return [max(min(t, L), L - (i * L) // (2 * b) - (i % 3)) for i in range(b)]


def _inverse_frequencies(case):
    """Turning speed of each pair in radians per position (64 bits), and the factor on cosine and sine.  factor > 1:
    the blend of interpolated and kept frequencies by wavelength, for a model trained to 4096 positions."""
    dim, theta, factor = case["rotary_dim"], case["theta"], case["factor"]
    kept = [theta ** (-2.0 * j / dim) for j in range(dim // 2)]
    if factor == 1.0:
        return kept, 1.0
    turns_at = lambda turns: dim * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    lo, hi = max(math.floor(turns_at(32.0)), 0), min(math.ceil(turns_at(1.0)), dim - 1)
    share = [min(max((j - lo) / max(hi - lo, 0.001), 0.0), 1.0) for j in range(dim // 2)]
    return [f / factor * s + f * (1.0 - s) for f, s in zip(kept, share)], 0.1 * math.log(factor) + 1.0


def _encode(x, code):
    """Codes and scales of rows: scale = largest magnitude / largest code, code = round(x * (largest code / largest
    magnitude))."""
    x = x.float()
    top = x.abs().amax(-1)
    scale = top / LARGEST[code]
    held = scale >= SMALLEST_SCALE
    per = torch.where(held, LARGEST[code] / top, torch.zeros_like(top))
    y = x * per[..., None]
    y = torch.round(y) if code == "int8" else y
    y = y.clamp(-LARGEST[code], LARGEST[code])
    return y.to(CODES[code]), torch.where(held, scale, torch.zeros_like(scale))


def _rows(g, case, length, kind):
    """Key or value rows (batch, kv_heads, length, head_dim) with what caches show: channels of unlike size and mean."""
    d = case["head_dim"]
    shape = (case["batch"], case["kv_heads"], length, d)
    size = torch.exp(0.5 * torch.randn(case["kv_heads"], 1, d, generator=g, device=DEVICE))
    mean = 0.5 * torch.randn(case["kv_heads"], 1, d, generator=g, device=DEVICE)
    return torch.randn(shape, generator=g, device=DEVICE).mul_(size).add_(mean).to(kind)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind = TYPES[case["type"]]
    b, d = case["batch"], case["head_dim"]
    s = {"case": case}
    if case["op"] == "rotary":
        n = case["tokens"]
        s["query"] = torch.randn(b, n, case["heads"], d, generator=g, device=DEVICE).to(kind).transpose(1, 2)
        s["key"] = torch.randn(b, n, case["kv_heads"], d, generator=g, device=DEVICE).to(kind).transpose(1, 2)
        freq, s["magnitude"] = _inverse_frequencies(case)
        s["inv_freq"] = torch.tensor(freq, dtype=torch.float64, device=DEVICE)
        s["position"] = (case["first"] + torch.randint(0, 1000, (b,), generator=g, device=DEVICE)).to(torch.int32)
        return s
    if case["op"] == "cache":
        n, cap, kv = case["tokens"], case["capacity"], case["kv_heads"]
        s["position"] = torch.randint(0, cap - n + 1, (b,), generator=g, device=DEVICE).to(torch.int32)
        if case["write"]:
            s["new_key"], s["new_value"] = _rows(g, case, n, kind), _rows(g, case, n, kind)
            for x in ("key", "value"):
                s[x + "_codes"] = torch.zeros(b, kv, cap, d, dtype=CODES[case["code"]], device=DEVICE)
                s[x + "_scales"] = torch.zeros(b, kv, cap, device=DEVICE)
        else:
            for x in ("key", "value"):
                s[x + "_codes"], s[x + "_scales"] = _encode(_rows(g, case, cap, kind), case["code"])
        return s
    n, L = case.get("tokens", 1), case["kv_len"]
    s["query"] = (1.5 * torch.randn(b, case["heads"], n, d, generator=g, device=DEVICE)).to(kind)
    s["kv_lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)
    for x in ("key", "value"):
        rows = _rows(g, case, L, kind)
        if case["code"] == "dense":
            s[x] = rows
        else:
            s[x + "_codes"], s[x + "_scales"] = _encode(rows, case["code"])
    if case["op"] == "tree":      # tree_mask[.., t, u]: drafted token t sees drafted token u, its ancestor or itself
        trees = 1 if case["shared_tree"] else b
        at = torch.arange(n, device=DEVICE)
        pick = torch.rand(trees, n, generator=g, device=DEVICE)
        parent = at - 1 - (pick * at.clamp(max=4)).long()      # one of the few tokens before
        see = torch.zeros(trees, n, n, dtype=torch.bool, device=DEVICE)
        for i in range(n):
            if i:
                see[:, i] = see[torch.arange(trees, device=DEVICE), parent[:, i]]
            see[:, i, i] = True
        s["tree_mask"] = see[0] if case["shared_tree"] else see
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------
def _turn(x, cos, sin, dim, interleaved):
    y = x.float()
    if interleaved:
        a, b = y[..., 0:dim:2], y[..., 1:dim:2]
        z = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :dim // 2], y[..., dim // 2:dim]
        z = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((z, y[..., dim:]), -1).to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    at = s["position"][:, None] + torch.arange(case["tokens"], device=DEVICE)
    angle = (at.double()[..., None] * s["inv_freq"])[:, None]
    cos, sin = (torch.cos(angle) * s["magnitude"]).float(), (torch.sin(angle) * s["magnitude"]).float()
    return [_turn(s[x], cos, sin, case["rotary_dim"], case["interleaved"]) for x in ("query", "key")]


def _plain_cache(s):
    case = s["case"]
    b, kv, n = case["batch"], case["kv_heads"], case["tokens"]
    at = (s["position"][:, None] + torch.arange(n, device=DEVICE)).long()[:, None, :].expand(b, kv, n)
    bi = torch.arange(b, device=DEVICE)[:, None, None].expand(b, kv, n)
    hi = torch.arange(kv, device=DEVICE)[None, :, None].expand(b, kv, n)

    def one(x):
        codes, scales = s[x + "_codes"], s[x + "_scales"]
        if case["write"]:
            c, scale = _encode(s["new_" + x], case["code"])
            codes.view(torch.int8)[bi, hi, at] = c.view(torch.int8)
            scales[bi, hi, at] = scale
        c = codes.view(torch.int8)[bi, hi, at].view(codes.dtype)
        return (c.float() * scales[bi, hi, at][..., None]).to(TYPES[case["type"]])

    return [one("key"), one("value")]


def _plain_attention(s):
    case = s["case"]
    b, h, kv, d, L = (case[x] for x in ("batch", "heads", "kv_heads", "head_dim", "kv_len"))
    n = case.get("tokens", 1)
    if case["code"] == "dense":
        k, v = s["key"].float(), s["value"].float()
    else:
        k = s["key_codes"].float() * s["key_scales"][..., None]
        v = s["value_codes"].float() * s["value_scales"][..., None]
    q = s["query"].float().reshape(b, kv, h // kv, n, d) * d ** -0.5
    score = torch.matmul(q.reshape(b, kv, -1, d), k.transpose(2, 3)).view(b, kv, h // kv, n, L)
    at = torch.arange(L, device=DEVICE)
    first = s["kv_lens"][:, None] - n                     # the cache row of drafted token 0
    see = (at < first)[:, None, :].expand(b, n, L)
    if "tree_mask" in s:
        drafted = at - first                              # (batch, kv_len)
        inside = (drafted >= 0) & (drafted < n)
        tree = s["tree_mask"].expand(b, n, n)
        see = see | (torch.gather(tree, 2, drafted.clamp(0, n - 1).long()[:, None, :].expand(b, n, L)) & inside[:, None, :])
    else:
        see = see | (at == first)[:, None, :]
    score = score.masked_fill(~see[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.view(b, kv, -1, L), v) / total.view(b, kv, -1, 1).clamp(min=1e-38)
    return out.view(b, h, n, d).to(s["query"].dtype)


def _own(s):
    import kernel_collections_b200 as K
    case = s["case"]
    if case["op"] == "rotary":
        return K.rotary_embedding(s["query"], s["key"], s["inv_freq"], s["position"], interleaved=case["interleaved"],
                                  magnitude=s["magnitude"])
    if case["op"] == "tree" and case["code"] == "dense":
        return K.group_query_attention_tree(s["query"], s["key"], s["value"], s["tree_mask"], kv_lens=s["kv_lens"])
    cache = K.QuantizedCache(s["key_codes"], s["key_scales"], s["value_codes"], s["value_scales"])
    if case["op"] == "cache":
        if case["write"]:
            K.quantized_cache_append(cache, s["new_key"], s["new_value"], s["position"])
        return K.quantized_cache_read(cache, s["position"], case["tokens"], dtype=TYPES[case["type"]])
    return K.group_query_attention_quantized(s["query"], cache, s.get("tree_mask"), kv_lens=s["kv_lens"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "rotary":
        return _plain_rotary(state)
    if op == "cache":
        return _plain_cache(state)
    return _plain_attention(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------
def work(case):
    size = 4 if case["type"] == "f32" else 2
    b, d, n = case["batch"], case["head_dim"], case.get("tokens", 1)
    if case["op"] == "rotary":
        values = b * n * (case["heads"] + case["kv_heads"]) * d
        return {"bytes": 2 * size * values + 4 * b + 4 * case["rotary_dim"],
                "flops": 3 * b * n * (case["heads"] + case["kv_heads"]) * case["rotary_dim"]}
    kv = case["kv_heads"]
    if case["op"] == "cache":
        rows = 2 * b * kv * n
        held = rows * (d + 4)
        return {"bytes": rows * d * size + held + (rows * d * size + held if case["write"] else 0), "flops": 2 * rows * d}
    lens = _lengths(case)
    row = 2 * d * size if case["code"] == "dense" else 2 * (d + 4)
    mask = (n * n if case["shared_tree"] else b * n * n) if case["op"] == "tree" else 0
    return {"bytes": kv * sum(lens) * row + 2 * b * case["heads"] * n * d * size + mask + 4 * b,
            "flops": 4 * case["heads"] * n * d * sum(lens)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    b, d, n = case["batch"], case["head_dim"], case.get("tokens", 1)
    if case["op"] == "rotary":
        out = []
        dim = case["rotary_dim"]
        pos = s["position"].double()[:, None] + torch.arange(n, device=DEVICE).double()
        unit = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device=DEVICE),
                           pos[:, None, :, None] * s["inv_freq"])                        # (batch, 1, tokens, dim / 2)
        for x in (s["query"], s["key"]):
            y = x.double().clone()
            i = torch.arange(dim // 2, device=DEVICE)
            one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + dim // 2)
            z = torch.complex(y[..., one], y[..., two]) * unit
            y[..., one], y[..., two] = z.real, z.imag
            out.append(y)
        return out
    if case["op"] == "cache":
        out = []
        for x in ("key", "value"):
            rows = []
            for i, p in enumerate(s["position"].tolist()):
                if case["write"]:
                    y = s["new_" + x][i].double()
                    step = y.abs().amax(-1, keepdim=True) / LARGEST[case["code"]]
                    y = torch.where(step > 0, y / step, torch.zeros_like(y))
                    if case["code"] == "int8":
                        y = torch.round(y)
                    else:                                   # 4 significant bits down to 2^-6, steps of 2^-9 below
                        grid = torch.exp2((torch.frexp(y.abs()).exponent - 4).clamp(min=-9).double())
                        y = torch.round(y / grid) * grid
                    rows.append(y * step)
                else:
                    c = s[x + "_codes"][i, :, p:p + n].double()
                    rows.append(c * s[x + "_scales"][i, :, p:p + n, None].double())
            out.append(torch.stack(rows))
        return out
    kv, h = case["kv_heads"], case["heads"]
    out = torch.zeros(b, h, n, d, dtype=torch.float64, device=DEVICE)
    for i, length in enumerate(s["kv_lens"].tolist()):
        for j in range(kv):
            if case["code"] == "dense":
                k, v = s["key"][i, j, :length].double(), s["value"][i, j, :length].double()
            else:
                k = s["key_codes"][i, j, :length].double() * s["key_scales"][i, j, :length, None].double()
                v = s["value_codes"][i, j, :length].double() * s["value_scales"][i, j, :length, None].double()
            heads = slice(j * (h // kv), (j + 1) * (h // kv))
            score = torch.einsum("gtd,ld->gtl", s["query"][i, heads].double(), k) / math.sqrt(d)
            if "tree_mask" in s:
                tree = s["tree_mask"] if s["tree_mask"].dim() == 2 else s["tree_mask"][i]
                start = max(length - n, 0)
                score[:, :, start:] = score[:, :, start:].masked_fill(~tree[:, n - (length - start):], -math.inf)
            out[i, heads] = torch.einsum("gtl,ld->gtd", torch.softmax(score, -1), v)
    return out
