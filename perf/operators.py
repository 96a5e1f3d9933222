"""The operators of a decode step that reads its weights, its cache and its logits once, as measurable cases.

Three operators, called one after another by a program that draws several samples of one prompt and lets drafted tokens
run ahead:

* ``product``: a matrix product of few rows whose weights are 4-bit codes with a scale (and a zero point) per group of
  ``group`` entries along the sum;
* ``attention``: attention of rows whose requests share the first ``prefix`` keys and values of the paged cache, one row a
  request (decode) or several (drafted tokens to verify);
* ``verify``: which drafted tokens are kept, by the target's and the draft's probabilities and given random numbers, and
  the token drawn behind them.

A case is a dict of an ``op`` and its sizes.  ``run`` with ``own`` False computes the operators by elementary torch
operations in 32 bits (64 for probabilities); with ``own`` True it calls the package.
"""
import math

import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
#: the chance of a draft of a ``verify`` case with draft probabilities to be kept, as the inputs below make it
KEPT = 0.5
#: the most operations of a drawn ``attention`` case: what the largest listed one takes
MOST = 3.5e10


def _attention(name, requests, prefix, own_keys, heads, kv_heads, dim, page=16, rows=1, groups=1, type="bfloat16"):
    c = {"op": "attention", "groups": groups, "requests": requests, "rows": rows, "prefix": prefix, "own_keys": own_keys,
         "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "type": type}
    return dict(c, name=name) if name else c


def _product(name, rows, k, n, group, zeros=False, type="bfloat16"):
    c = {"op": "product", "rows": rows, "k": k, "n": n, "group": group, "zeros": zeros, "type": type}
    return dict(c, name=name) if name else c


def _verify(name, requests, drafts, vocab, distribution=True, ragged=False):
    c = {"op": "verify", "requests": requests, "drafts": drafts, "vocab": vocab, "distribution": distribution, "ragged": ragged}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token: queries, keys and values of a layer of width 1536
        _product("product 1 row qkv", 1, 1536, 2304, 128),
        # a batch of eight tokens through the gate and up matrices of a layer of width 4096
        _product("product 8 rows gate up", 8, 4096, 28672, 128),
        # drafted tokens of eight requests against the whole vocabulary, small groups with zero points
        _product("product 40 rows head", 40, 4096, 131072, 64, zeros=True),
        # the 32-bit path at odd sizes: the last group and the last columns are not full
        _product("product 3 rows odd f32", 3, 2005, 5501, 32, zeros=True, type="float32"),
        # two samples of a short prompt, the first tokens: latency
        _attention("attention 2 samples", 2, 128, 16, 12, 3, 128),
        # sixteen samples of a long prompt
        _attention("attention 16 samples", 16, 4096, 512, 12, 3, 128),
        # a batch behind one long document
        _attention("attention 64 samples", 64, 32768, 1024, 32, 8, 128),
        # five tokens a request to verify, two prompts, a prefix that ends inside a page
        _attention("attention drafts", 8, 2003, 300, 24, 8, 64, page=32, rows=5, groups=2),
        # the 32-bit path
        _attention("attention f32", 4, 1000, 65, 12, 3, 64, type="float32"),
        # one request, four drafts
        _verify("verify 1 request", 1, 4, 32000),
        # a batch over a large vocabulary
        _verify("verify 64 requests", 64, 7, 131072),
        # drafts by arg-max (no distribution), of different number, an odd vocabulary
        _verify("verify arg-max drafts", 13, 5, 49153, distribution=False, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["product", "attention", "verify"])
    if op == "product":
        type = rng.choice(["bfloat16", "bfloat16", "float32"])
        rows = _log_int(rng, 1, 64)
        return _product(None, rows, _log_int(rng, 256, 8192), _log_int(rng, 256, 16384), rng.choice([32, 64, 128]),
                        rng.random() < 0.5, type)
    if op == "attention":
        type = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        heads, kv_heads = rng.choice([(12, 3), (24, 8), (32, 8), (8, 1), (4, 4)])
        groups = rng.choice([1, 1, 2, 3])
        if type == "float32":
            return _attention(None, _log_int(rng, 1, 8), _log_int(rng, 16, 2048), _log_int(rng, 8, 256), heads, kv_heads,
                              rng.choice([64, 96, 128]), rng.choice([16, 32, 64]), rng.choice([1, 1, 3]), groups, type)
        c = _attention(None, _log_int(rng, 1, 64 // groups), _log_int(rng, 16, 16384), _log_int(rng, 8, 1024), heads, kv_heads,
                       rng.choice([64, 96, 128]), rng.choice([16, 32, 64]), rng.choice([1, 1, 2, 5, 8]), groups, type)
        while work(c)["flops"] > MOST:
            c["prefix"] //= 2
        return c
    return _verify(None, _log_int(rng, 1, 64), rng.randint(1, 8), _log_int(rng, 1000, 131072), rng.random() < 0.7,
                   rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _chunks(dim, type):
    """16-byte chunks of a cache row, and the elements of one."""
    elements = 16 // torch.empty((), dtype=type).element_size()
    return dim // elements, elements


def _stored(positions, dim, type):
    """Where the cache keeps logical chunk c of the row of a position: chunk c XOR (position mod 8) where a row is a
    multiple of eight chunks, else (c + position) mod chunks."""
    chunks, _ = _chunks(dim, type)
    c = torch.arange(chunks, device=positions.device)
    p = positions[:, None]
    return c ^ (p & 7) if chunks % 8 == 0 else (c + p) % chunks


def _prepare_attention(case, g):
    type, dim, page, kvh = TYPES[case["type"]], case["dim"], case["page"], case["kv_heads"]
    groups, requests, rows, prefix = case["groups"], case["requests"], case["rows"], case["prefix"]
    total = groups * requests
    dev = g.device
    own_max = max(case["own_keys"], rows)
    lens = torch.randint(max(rows, own_max // 2), own_max + 1, (total,), generator=g, device=dev)
    full = prefix // page                                   # pages that all requests of a group share
    tail = -(-(prefix + own_max) // page) - full            # and those of a request's own
    heads_of = torch.randn((groups, prefix, 2, kvh, dim), generator=g, device=dev).to(type)
    behind = torch.randn((total, tail * page - (prefix - full * page), 2, kvh, dim), generator=g, device=dev).to(type)
    rest = torch.cat([heads_of[:, full * page:].repeat_interleave(requests, 0), behind], 1)

    def pages_of(x, first):                                 # (..., keys, 2, kvh, dim) -> stored pages [n, 2, kvh, page, dim]
        keys = x.shape[1]
        chunks, elements = _chunks(dim, type)
        at = _stored(torch.arange(first, first + keys, device=dev), dim, type)
        y = x.reshape(x.shape[0], keys, 2 * kvh, chunks, elements)
        index = at[None, :, None, :, None].expand(x.shape[0], keys, 2 * kvh, chunks, elements)
        y = torch.empty_like(y).scatter_(3, index, y)
        return y.reshape(-1, page, 2, kvh, dim).permute(0, 2, 3, 1, 4)

    stored = torch.cat([pages_of(heads_of[:, : full * page], 0), pages_of(rest, full * page)])
    where = torch.randperm(stored.shape[0] + 3, generator=g, device=dev)[: stored.shape[0]]
    plane = torch.zeros((stored.shape[0] + 3, 2, kvh, page, dim), dtype=type, device=dev)
    plane[where] = stored
    first = where[: groups * full].reshape(groups, full).repeat_interleave(requests, 0)
    table = torch.cat([first, where[groups * full:].reshape(total, tail)], 1).to(torch.int32).contiguous()
    positions = (prefix + lens[:, None] - rows + torch.arange(rows, device=dev)).reshape(-1).to(torch.int32)
    q = torch.randn((total * rows, case["heads"] * dim), generator=g, device=dev).to(type)
    s = {"q": q, "plane": plane, "table": table, "positions": positions}
    if own:
        from tiny_inference_server_b200.kernels.attention_plan import SharedPrefixPlan
        s["plan"] = SharedPrefixPlan([(prefix, [(f * requests + i, rows) for i in range(requests)]) for f in range(groups)],
                                     case["heads"], kvh, dev)
        s["out"] = torch.empty_like(q)
        s["fault"] = torch.zeros(4, dtype=torch.int32, device=dev)
    return s


def _prepare_product(case, g):
    k, n, group = case["k"], case["n"], case["group"]
    dev = g.device
    groups = -(-k // group)
    codes = torch.randn((k, n), generator=g, device=dev).mul_(2.8).add_(8).round_().clamp_(0, 15).to(torch.uint8)
    scales = (torch.rand((groups, n), generator=g, device=dev) * 0.006 + 0.004).to(torch.bfloat16)
    zeros = torch.randint(6, 11, (groups, n), generator=g, device=dev).to(torch.uint8) if case["zeros"] else None
    x = torch.randn((case["rows"], k), generator=g, device=dev).to(TYPES[case["type"]])
    s = {"x": x, "codes": codes, "scales": scales, "zeros": zeros}
    if own:
        from tiny_inference_server_b200.weights.w4 import pack_w4
        s["w"] = pack_w4(codes, scales, zeros, group)
        s["out"] = torch.empty((case["rows"], n), dtype=x.dtype, device=dev)
    return s


def _prepare_verify(case, g):
    n, k, v = case["requests"], case["drafts"], case["vocab"]
    dev = g.device
    logits = torch.randn((n, k + 1, v), generator=g, device=dev) * 3.0
    p = logits.softmax(-1)
    if case["distribution"]:
        noise = torch.randn((n, k, v), generator=g, device=dev)
        q = (logits[:, :k] + 1.5 * noise).softmax(-1)
        drafts = torch.multinomial(q.reshape(n * k, v), 1, generator=g).reshape(n, k).to(torch.int32)
    else:
        q, drafts = None, logits[:, :k].argmax(-1).to(torch.int32)
    lens = torch.randint(0, k + 1, (n,), generator=g, device=dev).to(torch.int32) if case["ragged"] else None
    u = torch.rand((n, k + 1), generator=g, device=dev)
    s = {"p": p, "q": q, "drafts": drafts, "u": u, "lens": lens}
    if own:
        s["tokens"] = torch.empty((n, k + 1), dtype=torch.int32, device=dev)
        s["accepted"] = torch.empty(n, dtype=torch.int32, device=dev)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"attention": _prepare_attention, "product": _prepare_product, "verify": _prepare_verify}[case["op"]](case, g)
    return dict(s, case=case)


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _plain_product(s):
    group, k = s["case"]["group"], s["case"]["k"]
    of = torch.arange(k, device=s["x"].device) // group
    zero = s["zeros"].float()[of] if s["zeros"] is not None else 8.0
    w = (s["codes"].float() - zero) * s["scales"].float()[of]
    return (s["x"].float() @ w).to(s["x"].dtype)


def _logical(x, positions, dim, type):
    """Stored rows (..., keys, dim) back in the order of their elements."""
    chunks, elements = _chunks(dim, type)
    at = _stored(positions, dim, type)[..., None].expand(-1, -1, elements)
    y = x.reshape(*x.shape[:-1], chunks, elements)
    return y.gather(-2, at.expand(y.shape)).reshape(x.shape)


def _plain_attention(s):
    case = s["case"]
    type, dim, page, kvh = TYPES[case["type"]], case["dim"], case["page"], case["kv_heads"]
    groups, requests, rows, prefix = case["groups"], case["requests"], case["rows"], case["prefix"]
    total, g = groups * requests, case["heads"] // kvh
    dev = s["q"].device
    scale = 1.0 / math.sqrt(dim)
    q = s["q"].float() * scale
    table = s["table"].long()
    # the shared keys, once for all rows of a group
    pages = -(-prefix // page)
    at = torch.arange(pages * page, device=dev)
    shared = s["plane"][table[::requests, :pages]]                             # groups, pages, 2, kvh, page, dim
    shared = shared.permute(0, 2, 3, 1, 4, 5).reshape(groups, 2, kvh, pages * page, dim)
    shared = _logical(shared, at, dim, type)[..., :prefix, :].float()
    qs = q.reshape(groups, requests * rows, kvh, g, dim).permute(0, 2, 1, 3, 4).reshape(groups, kvh, requests * rows * g, dim)
    a = qs @ shared[:, 0].transpose(-1, -2)
    # every request's own keys behind them
    width = table.shape[1] * page - prefix
    at = torch.arange(prefix, prefix + width, device=dev)
    mine = s["plane"].permute(0, 3, 1, 2, 4)[table[:, at // page], at % page]    # total, width, 2, kvh, dim
    mine = _logical(mine.permute(0, 2, 3, 1, 4), at, dim, type).float()        # total, 2, kvh, width, dim
    qo = q.reshape(total, rows, kvh, g, dim).permute(0, 2, 1, 3, 4).reshape(total, kvh, rows * g, dim)
    b = qo @ mine[:, 0].transpose(-1, -2)
    seen = at[None, None, :] <= s["positions"].reshape(total, rows)[:, :, None]
    b = b.masked_fill(~seen.repeat_interleave(g, 1)[:, None], float("-inf"))
    # one softmax over both
    a = a.reshape(groups, kvh, requests, rows * g, prefix).permute(0, 2, 1, 3, 4).reshape(total, kvh, rows * g, prefix)
    top = torch.maximum(a.amax(-1, keepdim=True), b.amax(-1, keepdim=True))
    a, b = (a - top).exp(), (b - top).exp()
    norm = a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True)
    a = a.reshape(groups, requests, kvh, rows * g, prefix).permute(0, 2, 1, 3, 4).reshape(groups, kvh, requests * rows * g, prefix)
    o = (a @ shared[:, 1]).reshape(groups, kvh, requests, rows * g, dim).permute(0, 2, 1, 3, 4).reshape(total, kvh, rows * g, dim)
    o = (o + b @ mine[:, 1]) / norm
    return o.reshape(total, kvh, rows, g, dim).permute(0, 2, 1, 3, 4).reshape(total * rows, kvh * g * dim).to(type)


def _mass(x):
    """Probabilities in 64 bits; what is not a positive number counts as zero."""
    x = x.double()
    return torch.where((x > 0) & (x < float("inf")), x, 0.0)


def _plain_verify(s):
    p, q, u = s["p"], s["q"], s["u"].double()
    n, k, v = p.shape[0], p.shape[1] - 1, p.shape[2]
    dev = p.device
    lens = s["lens"].long() if s["lens"] is not None else torch.full((n,), k, device=dev)
    drafts = s["drafts"].long()
    real = (drafts >= 0) & (drafts < v)
    at = torch.where(real, drafts, 0)[..., None]
    target = torch.where(real, _mass(p[:, :k].gather(2, at)[..., 0]), 0.0)
    draft = _mass(q.gather(2, at)[..., 0]) if q is not None else torch.ones_like(target)
    kept = (u[:, :k] * draft < target) & (torch.arange(k, device=dev) < lens[:, None])
    accepted = kept.long().cumprod(1).sum(1)
    each = torch.arange(n, device=dev)
    row = _mass(p[each, accepted])
    last = accepted.clamp(max=k - 1)
    if q is not None:
        other = _mass(q[each, last])
    else:
        other = torch.zeros_like(row).scatter_(1, at[each, last], real[each, last].double()[:, None])
    left = (row - torch.where((accepted < lens)[:, None], other, 0.0)).clamp(min=0)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, row)
    sums = left.cumsum(1)
    index = torch.arange(v, device=dev)
    beyond = torch.where(sums > u[:, k:] * sums[:, -1:], index, v).amin(1)
    token = torch.where(beyond < v, beyond, torch.where(left > 0, index, -1).amax(1))
    places = torch.arange(k + 1, device=dev)
    tokens = torch.where(places < accepted[:, None], torch.cat([drafts, drafts[:, :1]], 1), -1)
    tokens = torch.where(places == accepted[:, None], token[:, None], tokens)
    return tokens.to(torch.int32), accepted.to(torch.int32)


def run(s):
    op = s["case"]["op"]
    if own:
        from tiny_inference_server_b200.kernels import ops
        if op == "product":
            return ops.gemm_w4(s["x"], s["w"], s["out"])
        if op == "attention":
            case = s["case"]
            return ops.shared_prefix_attention(s["q"], s["out"], s["plane"], s["table"], s["positions"], s["plan"], s["fault"],
                                               max_position=case["prefix"] + max(case["own_keys"], case["rows"]) - 1)
        return ops.verify_drafts(s["p"], s["q"], s["drafts"], s["u"], s["lens"], s["tokens"], s["accepted"])
    return {"product": _plain_product, "attention": _plain_attention, "verify": _plain_verify}[op](s)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    if case["op"] == "product":
        rows, k, n, groups = case["rows"], case["k"], case["n"], -(-case["k"] // case["group"])
        size = 4 if case["type"] == "float32" else 2
        return {"bytes": k * n / 2 + groups * n * (3 if case["zeros"] else 2) + rows * (k + n) * size, "flops": 2.0 * rows * k * n}
    if case["op"] == "attention":
        size = 4 if case["type"] == "float32" else 2
        rows = case["groups"] * case["requests"] * case["rows"]
        own_keys = 0.75 * max(case["own_keys"], case["rows"])              # a request's own keys, on average
        keys = case["groups"] * (case["prefix"] + case["requests"] * own_keys)
        return {"bytes": size * (2 * keys * case["kv_heads"] * case["dim"] + 2 * rows * case["heads"] * case["dim"]),
                "flops": 4.0 * rows * case["heads"] * case["dim"] * (case["prefix"] + own_keys)}
    n, k, v = case["requests"], case["drafts"], case["vocab"]
    rows = 1 + (1 - KEPT ** k if case["distribution"] else 0)              # the target's row, and the draft's behind a rejection
    return {"bytes": n * (rows * v * 4 + k * 16 + 4 + (k + 2) * 4), "flops": n * rows * v}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "verify":
        return None                                         # whole numbers
    s = prepare(case, seed)
    if case["op"] == "product":
        k, n, group = case["k"], case["n"], case["group"]
        y = torch.zeros((case["rows"], n), dtype=torch.float64, device=s["x"].device)
        for i, a in enumerate(range(0, k, group)):
            z = s["zeros"][i].double() if s["zeros"] is not None else 8.0
            y += (s["x"][:, a:a + group].double() @ (s["codes"][a:a + group].double() - z)) * s["scales"][i].double()
        return y
    type, dim, page, kvh, h = TYPES[case["type"]], case["dim"], case["page"], case["kv_heads"], case["heads"]
    rows, q = case["rows"], s["q"].double().reshape(-1, h, dim)
    chunks, elements = _chunks(dim, type)
    outs = []
    for r in range(case["groups"] * case["requests"]):
        at = [int(x) for x in s["positions"][r * rows:(r + 1) * rows]]
        keys = at[-1] + 1
        pool = s["plane"][s["table"][r, : -(-keys // page)].long()].transpose(0, 2).transpose(0, 1)     # 2, kvh, pages, page, dim
        flat = pool.reshape(2, kvh, -1, chunks, elements)[:, :, :keys]
        pos = torch.arange(keys, device=q.device)[:, None]
        c = torch.arange(chunks, device=q.device)[None]
        place = torch.bitwise_xor(c, pos % 8) if chunks % 8 == 0 else torch.remainder(c + pos, chunks)
        kv = flat[:, :, pos.expand(keys, chunks), place].reshape(2, kvh, keys, dim).double()
        for j in range(rows):
            x = q[r * rows + j].reshape(kvh, h // kvh, dim)
            w = torch.softmax(torch.einsum("kgd,ktd->kgt", x, kv[0, :, : at[j] + 1]) / dim ** 0.5, -1)
            outs.append(torch.einsum("kgt,ktd->kgd", w, kv[1, :, : at[j] + 1]).reshape(1, h * dim))
    return torch.cat(outs)
