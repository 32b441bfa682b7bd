"""The serving operators around the paged key/value cache, as cases that can be timed.

* ``append``: rotary embedding of a ragged batch of new tokens and the write of their keys and values into the
  pages of the cache.
* ``packed``: causal grouped-query attention over whole prompts of different lengths, packed one after another.
* ``paged``: causal grouped-query attention of new tokens (one or a chunk of them a sequence) over the paged cache.

``run`` computes them in elementary torch operations, or, where ``own`` is true, through the package's entry points.
"""
import importlib
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_GGML = {"f32": 0, "f16": 1, "bf16": 30}
_ROPE_BASE = 1e6


def _append(name, type, heads, kv_heads, head_dim, sequences, q_min, q_max, kv_min, kv_max, page, layout, lengths):
    return {"name": name, "op": "append", "type": type, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "sequences": sequences, "q_min": q_min, "q_max": q_max, "kv_min": kv_min, "kv_max": kv_max, "page": page,
            "layout": layout, "lengths": lengths}


def _paged(*a):
    return dict(_append(*a), op="paged")


def _packed(name, type, heads, kv_heads, head_dim, sequences, q_min, q_max, pad, lengths):
    return {"name": name, "op": "packed", "type": type, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "sequences": sequences, "q_min": q_min, "q_max": q_max, "pad": pad, "lengths": lengths}


def listed():
    return [
        # a decode step's append of eight chats with a small model: launch latency is what counts
        _append("append decode f32", "f32", 14, 2, 64, 8, 1, 1, 64, 1280, 16, "position", 1),
        # the prompts of several requests of a larger model entering the cache at once
        _append("append prompts bf16", "bf16", 28, 4, 128, 9, 300, 2400, 300, 6000, 64, "head", 2),
        # one long document
        _packed("packed one bf16", "bf16", 28, 4, 128, 1, 8192, 8192, 0, 3),
        # a batch of prompts of very different lengths with a small model, the buffer longer than what is in it
        _packed("packed ragged bf16", "bf16", 14, 2, 64, 13, 17, 4000, 77, 4),
        # many short questions, single tokens among them: few keys for each row
        _packed("packed short f16", "f16", 32, 8, 128, 61, 1, 64, 3, 5),
        # the framework's own 32-bit activations, prompts of a small model
        _packed("packed f32", "f32", 14, 2, 64, 3, 400, 2000, 0, 6),
        # one chat's decode step with a small model: latency
        _paged("decode one f32", "f32", 14, 2, 64, 1, 1, 1, 1280, 1280, 16, "position", 7),
        # a serving step: chats of all ages
        _paged("decode 64 bf16", "bf16", 28, 4, 128, 64, 1, 1, 16, 8192, 64, "position", 8),
        # one chat over a very long context
        _paged("decode long f16", "f16", 32, 8, 128, 1, 1, 1, 131071, 131071, 256, "head", 9),
        # a full machine
        _paged("decode 256 bf16", "bf16", 28, 4, 128, 256, 1, 1, 1024, 8000, 128, "head", 10),
        # a chunk of a long prompt over what is cached of it
        _paged("chunk bf16", "bf16", 28, 4, 128, 1, 1000, 1000, 32700, 32700, 16, "position", 11),
        # chunks of some requests beside single tokens of others, 32-bit activations over a 16-bit cache
        _paged("mixed f32", "f32", 14, 2, 64, 16, 1, 256, 256, 4096, 32, "position", 12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    op = rng.choice(["append", "packed", "packed", "paged", "paged", "paged"])
    heads, kv_heads, head_dim = rng.choice([(14, 2, 64), (28, 4, 128), (32, 8, 128), (8, 8, 64), (16, 1, 64), (10, 2, 128), (9, 3, 64),
                                            (12, 4, 128)])
    type = rng.choice(["f32", "f16", "bf16"])
    lengths = rng.randrange(1 << 30)
    if op == "packed":
        # the cost of the plain form goes with the square of all tokens
        most = 7000 * 28 // max(28, heads) if type != "f32" else 3500
        total = _log(rng, 64, most)
        n = _log(rng, 1, min(64, total))
        return dict(_packed("", type, heads, kv_heads, head_dim, n, 1 if n > 2 else max(1, total // n // 3), max(1, total // n),
                            rng.choice([0, 0, 1, 50]), lengths))
    page, layout = rng.choice([16, 32, 64, 128, 256]), rng.choice(["position", "head"])
    if op == "append":
        n, longest = _log(rng, 1, 128), _log(rng, 1, 64)
        return _append("", type, heads, kv_heads, head_dim, n, 1, longest, longest, longest + _log(rng, 1, 8000), page, layout, lengths)
    if rng.random() < 0.6:  # single tokens (a few, as where a draft is verified)
        n = _log(rng, 1, 192)
        longest = rng.choice([1, 1, 1, 2, 4, 5])
        kv = _log(rng, 16, min(120000, 1000000 // n))
        return _paged("", type, heads, kv_heads, head_dim, n, 1, longest, longest, longest + kv, page, layout, lengths)
    n = _log(rng, 1, 12)
    longest = _log(rng, 8, 1000 // n + 8)
    kv = _log(rng, 16, 20000 // n)
    return _paged("", type, heads, kv_heads, head_dim, n, rng.choice([1, longest]), longest, longest, longest + kv, page, layout, lengths)


def _shape(case):
    """(new tokens, cached positions) of each sequence, from the case alone."""
    rng = np.random.default_rng(case["lengths"])
    n = case["sequences"]

    def spread(lo, hi):  # even over the logarithm
        return np.clip(np.rint(np.exp(rng.uniform(math.log(lo), math.log(hi + 0.49), n))), lo, hi).astype(np.int64)

    new = spread(case["q_min"], case["q_max"])
    if case["op"] == "packed":
        return new, new
    return new, np.maximum(new, spread(case["kv_min"], case["kv_max"]))


def _cache_type(case):
    return "bf16" if case["type"] == "bf16" else "f16"


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    new, kv = _shape(case)
    h, hk, d, n = case["heads"], case["kv_heads"], case["head_dim"], case["sequences"]
    t = _TYPES[case["type"]]
    used = int(new.sum())
    tokens = used + case.get("pad", 0)
    # rows as the joint projection leaves them: [q | k | v]; keys stand off zero by a bias of their channel
    rows = torch.randn(tokens, (h + 2 * hk) * d, generator=g, device="cuda")
    rows[:, h * d:(h + hk) * d] += torch.randn(hk * d, generator=g, device="cuda")
    rows = rows.to(t)
    start = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
    st = {"case": case, "used": used, "tokens": tokens, "rows": rows, "start": start, "out": torch.zeros(tokens, h * d, dtype=t, device="cuda"),
          "q": rows[:, :h * d], "k": rows[:, h * d:(h + hk) * d], "v": rows[:, (h + hk) * d:]}
    if case["op"] != "packed":
        page = case["page"]
        pages = (kv + page - 1) // page
        width, spare = int(pages.max()) + 1, 3
        count = int(pages.sum()) + spare
        order = torch.randperm(count, generator=g, device="cuda").to(torch.int32)
        first = torch.from_numpy(np.concatenate([[0], np.cumsum(pages)])[:-1].astype(np.int64)).cuda()
        at = torch.arange(width, device="cuda")
        at = torch.where(at[None, :] < torch.from_numpy(pages).cuda()[:, None], first[:, None] + at[None, :], 0)
        st["table"] = order[at].contiguous()
        st["length"] = torch.from_numpy(kv.astype(np.int32)).cuda()
        ct = _TYPES[_cache_type(case)]
        shape = (count, hk, page, d) if case["layout"] == "head" else (count, page, hk, d)
        bias = torch.randn(hk, d, generator=g, device="cuda")
        bias = bias[:, None, :] if case["layout"] == "head" else bias
        st["keys"] = torch.randn(shape, generator=g, device="cuda", dtype=ct).add_(bias.to(ct))
        st["values"] = torch.randn(shape, generator=g, device="cuda", dtype=ct)
        st["longest"] = int(new.max())
        st["reach"] = int(kv.max())
    if own:
        st["package"] = p = importlib.import_module("my-inference-engine_b200")
        if case["op"] != "packed":
            s = (hk * page * d, d, page * d) if case["layout"] == "head" else (page * hk * d, hk * d, d)
            st["cache"] = p.PagedCache(st["keys"], st["values"], _GGML[_cache_type(case)], hk, d, page, count, page_stride=s[0],
                                       position_stride=s[1], head_stride=s[2])
            st["batch"] = p.PagedBatch(start, st["length"], st["table"], n, tokens, width, max_query=st["longest"])
    return st


def _run_own(st):
    c, p = st["case"], st["package"]
    h, hk, d, t = c["heads"], c["kv_heads"], c["head_dim"], _GGML[c["type"]]
    ld = (h + 2 * hk) * d
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "packed":
        p.packed_attention(t, h, hk, d, st["start"], c["sequences"], st["tokens"], st["q"], ld, st["k"], ld, st["v"], ld, st["out"], h * d,
                           stream=stream)
        return st["out"]
    if c["op"] == "append":
        p.paged_append(st["cache"], st["batch"], t, h, st["q"], ld, st["k"], ld, st["v"], ld, rope_base=_ROPE_BASE, q_out=st["out"],
                       q_out_ld=h * d, stream=stream)
        return {"q": st["out"], "keys": st["keys"], "values": st["values"]}
    p.paged_attention(st["cache"], st["batch"], t, h, st["q"], ld, st["out"], h * d, stream=stream)
    return st["out"]


def _sequence_of(st):
    """The sequence of each token and its place among that sequence's new tokens."""
    i = torch.arange(st["used"], device="cuda")
    s = torch.searchsorted(st["start"][1:].long(), i, right=True)
    return s, i - st["start"].long()[s]


def _softmax_(s):
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    s /= s.sum(-1, keepdim=True)
    return s


def _plain_packed(st):
    c, n = st["case"], st["used"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    seq, _ = _sequence_of(st)
    i = torch.arange(n, device="cuda")
    hidden = (seq[:, None] != seq[None, :]) | (i[:, None] < i[None, :])
    q = (st["q"][:n].float() / math.sqrt(d)).view(n, hk, h // hk, d).permute(1, 2, 0, 3).reshape(hk, h // hk * n, d)
    k = st["k"][:n].float().view(n, hk, d).permute(1, 2, 0)
    v = st["v"][:n].float().view(n, hk, d).transpose(0, 1)
    s = torch.matmul(q, k).view(hk, h // hk, n, n).masked_fill_(hidden, -math.inf)
    o = torch.matmul(_softmax_(s).view(hk, h // hk * n, n), v).view(hk, h // hk, n, d)
    st["out"][:n] = o.permute(2, 0, 1, 3).reshape(n, h * d)
    return st["out"]


def _plain_append(st):
    c, n = st["case"], st["used"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    seq, i = _sequence_of(st)
    start, length = st["start"].long(), st["length"].long()
    position = length[seq] - (start[seq + 1] - start[seq]) + i
    angle = position.double()[:, None] * torch.pow(_ROPE_BASE, -2.0 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]

    def turned(x, heads):
        a, b = x[:n].float().view(n, heads, 2, d // 2).unbind(2)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    page, row = st["table"].long()[seq, position // c["page"]], position % c["page"]
    keys, values = (x.transpose(1, 2) if c["layout"] == "head" else x for x in (st["keys"], st["values"]))
    keys[page, row] = turned(st["k"], hk).to(keys.dtype)
    values[page, row] = st["v"][:n].view(n, hk, d).to(values.dtype)
    st["out"][:n] = turned(st["q"], h).view(n, h * d).to(st["out"].dtype)
    return {"q": st["out"], "keys": st["keys"], "values": st["values"]}


def _plain_paged(st):
    c, n = st["case"], st["used"]
    h, hk, d, m = c["heads"], c["kv_heads"], c["head_dim"], c["sequences"]
    reach, longest = st["reach"], st["longest"]
    seq, i = _sequence_of(st)
    j = torch.arange(reach, device="cuda")
    page, row = st["table"].long()[:, j // c["page"]], j % c["page"]
    keys, values = (x.transpose(1, 2) if c["layout"] == "head" else x for x in (st["keys"], st["values"]))
    k = keys[page, row].permute(0, 2, 3, 1).float()  # sequences x kv_heads x head_dim x positions
    v = values[page, row].transpose(1, 2).float()
    q = torch.zeros(m, longest, h * d, device="cuda")
    q[seq, i] = st["q"][:n].float() / math.sqrt(d)
    q = q.view(m, longest, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(m, hk, h // hk * longest, d)
    start, length = st["start"].long(), st["length"].long()
    last = length[:, None] - (start[1:] - start[:-1])[:, None] + torch.arange(longest, device="cuda")
    hidden = j[None, None, :] > torch.minimum(last, length[:, None] - 1)[:, :, None]
    s = torch.matmul(q, k).view(m, hk, h // hk, longest, reach).masked_fill_(hidden[:, None, None], -math.inf)
    o = torch.matmul(_softmax_(s).view(m, hk, h // hk * longest, reach), v)
    o = o.view(m, hk, h // hk, longest, d).permute(0, 3, 1, 2, 4).reshape(m, longest, h * d)
    st["out"][:n] = o[seq, i].to(st["out"].dtype)
    return st["out"]


def run(state):
    if own:
        return _run_own(state)
    return {"packed": _plain_packed, "append": _plain_append, "paged": _plain_paged}[state["case"]["op"]](state)


def work(case):
    new, kv = _shape(case)
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    size, cached = _TYPES[case["type"]].itemsize, _TYPES[_cache_type(case)].itemsize
    tokens = int(new.sum())
    pairs = int((new * kv - new * (new - 1) // 2).sum())
    if case["op"] == "append":
        return {"bytes": tokens * d * (2 * h * size + 2 * hk * (size + cached)), "flops": tokens * d * 3 * (h + hk)}
    bytes = 2 * tokens * h * d * size
    bytes += 2 * tokens * hk * d * size if case["op"] == "packed" else 2 * int(kv.sum()) * hk * d * cached
    return {"bytes": bytes, "flops": 4 * d * h * pairs}


def exact(case, seed):
    """One sequence and one head of keys after another, in 64 bits."""
    st = prepare(case, seed)
    new, kv = _shape(case)
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    group = h // hk
    out = st["out"].double()
    q = st["q"].double().view(-1, h, d)
    if case["op"] == "append":
        q_out, keys, values = out.view(-1, h, d), st["keys"].double(), st["values"].double()
        turn = torch.exp(-math.log(_ROPE_BASE) * torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    k_new, v_new = (st[x].double().view(-1, hk, d) for x in ("k", "v"))
    t0 = 0
    for s in range(case["sequences"]):
        length, upto = int(new[s]), int(kv[s])
        mine = slice(t0, t0 + length)
        t0 += length
        if case["op"] == "append":
            at = torch.arange(upto - length, upto, device="cuda")
            unit = torch.polar(torch.ones(length, d // 2, device="cuda", dtype=torch.float64), at.double()[:, None] * turn[None, :])[:, None]

            def rotate(x):
                z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * unit
                return torch.cat([z.real, z.imag], -1)

            q_out[mine] = rotate(q[mine])
            where = st["table"][s].long()[torch.div(at, case["page"], rounding_mode="floor")]
            if case["layout"] == "head":
                keys[where, :, at % case["page"]] = rotate(k_new[mine])
                values[where, :, at % case["page"]] = v_new[mine]
            else:
                keys[where, at % case["page"]] = rotate(k_new[mine])
                values[where, at % case["page"]] = v_new[mine]
            continue
        if case["op"] == "paged":
            pages = st["table"][s].long()[:-(-upto // case["page"])]
            ks, vs = st["keys"][pages], st["values"][pages]
            if case["layout"] == "head":
                ks, vs = ks.permute(0, 2, 1, 3), vs.permute(0, 2, 1, 3)
            ks, vs = (x.reshape(-1, hk, d)[:upto].double() for x in (ks, vs))
        else:
            ks, vs = k_new[mine], v_new[mine]
        allowed = torch.ones(length, upto, device="cuda", dtype=torch.bool).tril(upto - length)
        for b in range(hk):
            for a in range(b * group, (b + 1) * group):
                logits = torch.where(allowed, q[mine, a] @ ks[:, b].T / math.sqrt(d), -math.inf)
                w = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
                out[mine, a * d:(a + 1) * d] = w @ vs[:, b]
    return {"q": out, "keys": keys, "values": values} if case["op"] == "append" else out
