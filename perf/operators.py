"""Cases of the serving operators: the paged key/value cache (append, read back), attention of a
ragged batch over it, and sampling from given random numbers.

``run`` computes a case in plain torch operations, or with ``own`` set through
``parrot_b200.bridge``.  Shapes are Parrot XL's (8 query and 2 key/value heads of 96, window 2048,
128-wide latent, 4096 positions, 32768 tokens of vocabulary), the tiny configuration's and a few
generic ones.

A batch is ragged: row ``query_start[b] + i`` of the packed projection is token ``i`` of sequence
``b``, at position ``context_len[b] - (query_start[b + 1] - query_start[b]) + i``; position ``p`` of
sequence ``b`` is row ``p % page`` of page ``page_table[b, p // page]`` in pools
``[pages, kv heads, page, head width]``.  An 8-bit pool holds e4m3 numbers and, for each row of
each head, one byte ``s``: the row's values are ``number * 2 ** (s - 127)``.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_DEV = "cuda"
_E4M3 = torch.float8_e4m3fn
#: the exponents that a row's scale may take: every scaled number is a normal bf16
_MIN_EXP, _MAX_EXP = -110, 119
_NEG = float("-inf")

_LOCAL = {"heads": 8, "kv_heads": 2, "width": 96}      # Parrot XL's sliding-window layers
_LATENT = {"heads": 8, "kv_heads": 1, "width": 128}    # its absorbed latent layers: keys = values


def _bridge():
    root = str(Path(__file__).resolve().parent.parent / "parrot-h200-worker_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from parrot_b200 import bridge
    return bridge


# ---------------------------------------------------------------------------------------- cases
def _attend(name, shape, *, latent=False, queries, contexts, page, dtype, window, sinks):
    return {"name": name, "op": "attend", **shape, "latent": latent, "queries": queries,
            "contexts": contexts, "page": page, "dtype": dtype, "window": window, "sinks": sinks}


def listed():
    return [
        # a decode step's new rows of eight sequences into the cache: the smallest call
        {"name": "append decode 8 bf16", "op": "append", **_LOCAL, "latent": False,
         "queries": "1*8", "contexts": "129,4096,1,700,2048,2049,63,64", "page": 64,
         "dtype": "bf16"},
        # prompts written in 8 bits, then read back as the dense cache that decoding replays on
        {"name": "append and read e4m3", "op": "append", **_LOCAL, "latent": False,
         "queries": "512,33,1,1000,128,257", "contexts": "512,33,1,1000,128,257", "page": 32,
         "dtype": "e4m3"},
        # a full 8-bit cache read back
        {"name": "read e4m3 8", "op": "read", **_LOCAL, "latent": False,
         "queries": "1*8", "contexts": "4096,4095,1,2049,3000,17,640,4096", "page": 64,
         "dtype": "e4m3"},
        # a latent cache read back
        {"name": "read latent bf16", "op": "read", **_LATENT, "latent": True,
         "queries": "1*16", "contexts": "4096*8,129,128,127,1,2500,2048,333,4000", "page": 128,
         "dtype": "bf16"},
        # one decode step of one sequence, where latency counts
        _attend("decode 1 bf16", _LOCAL, queries="1", contexts="4096", page=64, dtype="bf16",
                window=2048, sinks=0),
        # a decode step of a full batch on an 8-bit cache, with sinks
        _attend("decode 64 e4m3 sinks", _LOCAL, queries="1*64",
                contexts="4096*20,2048*8,129*8,1,2,3000*10,511,512,513,1500*13", page=64,
                dtype="e4m3", window=2048, sinks=4),
        # a prompt of 512 tokens
        _attend("chunk 512 bf16", _LOCAL, queries="512", contexts="512", page=64, dtype="bf16",
                window=2048, sinks=0),
        # latent layers: chunks behind long contexts
        _attend("chunk latent 4", _LATENT, latent=True, queries="256,256,100,256",
                contexts="4096,1000,100,2500", page=64, dtype="bf16", window=0, sinks=0),
        # continuous batching: decode rows beside chunks, 8-bit cache, sinks
        _attend("mixed e4m3 sinks", _LOCAL, queries="1,1,700,1,129,512",
                contexts="4096,513,4000,1,129,2600", page=32, dtype="e4m3", window=2048, sinks=4),
        # four whole prompts of 4096 tokens: the largest
        _attend("prefill 4x4096 bf16", _LOCAL, queries="4096*4", contexts="4096*4", page=64,
                dtype="bf16", window=2048, sinks=0),
        # one row of logits, top-p only
        {"name": "sample 1", "op": "sample", "rows": 1, "vocab": 32768, "mix": "top_p"},
        # a decode batch whose rows all ask for something else
        {"name": "sample 64", "op": "sample", "rows": 64, "vocab": 32768, "mix": "all"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "attend", "sample"])
    if op == "sample":
        return {"op": op, "rows": _log(rng, 1, 256), "vocab": rng.choice([32768, 4096, 50257, _log(rng, 100, 131072)]),
                "mix": rng.choice(["all", "none", "top_k", "top_p", "min_p", "greedy"])}
    latent = rng.random() < 0.25
    shape = dict(_LATENT) if latent else dict(rng.choice(
        [_LOCAL, _LOCAL, _LOCAL, {"heads": 4, "kv_heads": 2, "width": 32},
         {"heads": 12, "kv_heads": 4, "width": 64}, {"heads": 4, "kv_heads": 4, "width": 128}]))
    page, dtype = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "e4m3"])
    kind = rng.choice(["decode", "few", "chunk", "mixed"])
    most = 32768 if kind == "decode" else 8192
    budget = 1 << 25  # query heads x queries x keys, rounded up to the longest of each
    while True:
        n = _log(rng, 1, 64 if kind in ("decode", "few") else 8)
        q = [1 if kind == "decode" or (kind == "mixed" and rng.random() < 0.5)
             else rng.randint(1, 8) if kind == "few" else _log(rng, 9, 2048) for _ in range(n)]
        c = [min(most, x + (_log(rng, 1, most) if rng.random() < 0.8 else 0)) for x in q]
        if n * max(q) * max(c) <= budget and n * max(c) <= 1 << 18:
            break
    case = {"op": op, **shape, "latent": latent, "queries": ",".join(map(str, q)),
            "contexts": ",".join(map(str, c)), "page": page, "dtype": dtype}
    if op == "attend":
        case["window"] = 0 if latent else rng.choice([0, 2048, 2048, _log(rng, 1, 4096)])
        case["sinks"] = rng.choice([0, 0, 4, rng.randint(1, 200)]) if case["window"] else 0
    return case


def _lengths(text):
    out = []
    for part in text.split(","):
        value, _, times = part.partition("*")
        out += [int(value)] * int(times or 1)
    return out


# --------------------------------------------------------------------------------------- inputs
def _scale_exponents(amax):
    """The least ``e`` with ``amax <= 448 * 2**e``, clamped (448 = 1.75 * 2**8)."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > 0.875).to(x.dtype)
    return torch.where(amax > 0, e, _MIN_EXP).clamp(_MIN_EXP, _MAX_EXP)


def _quantised(x):
    """fp32 or fp64 rows -> (e4m3 numbers, scale bytes)."""
    e = _scale_exponents(x.abs().amax(-1))
    return torch.ldexp(x, -e[..., None]).to(_E4M3), (e + 127).to(torch.uint8)


def _values(numbers, scale, dtype):
    x = numbers.to(dtype)
    return x if scale is None else torch.ldexp(x, scale.to(torch.int32)[..., None] - 127)


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=_DEV)

    if case["op"] == "sample":
        rows, vocab, mix = case["rows"], case["vocab"], case["mix"]
        i = torch.arange(rows, device=_DEV)

        def param(values, off, dtype):
            v = torch.tensor(values, device=_DEV, dtype=dtype)
            return v[i % len(values)] if mix == "all" or off else torch.full((rows,), values[0], device=_DEV, dtype=dtype)

        return {
            "op": "sample",
            # a language model's logits: wide, with some tokens that stand out
            "logits": (2.5 * normal(rows, vocab) + 4.0 * (normal(rows, vocab) > 3.0)).to(torch.bfloat16),
            "uniform": torch.rand(rows, generator=gen, device=_DEV),
            "temperature": param([0.0] if mix == "greedy" else [0.8, 1.0, 0.0, 1.3, 0.6], mix != "greedy", torch.float32),
            "top_k": param([0, 50, 1, 1000, 7] if mix == "all" else [40] if mix == "top_k" else [0], False, torch.int32),
            "top_p": param([0.9, 1.0, 0.95, 0.5] if mix == "all" else [0.9] if mix == "top_p" else [1.0], False, torch.float32),
            "min_p": param([0.0, 0.05, 0.0] if mix == "all" else [0.02] if mix == "min_p" else [0.0], False, torch.float32),
        }

    heads, kv_heads, width, page = case["heads"], case["kv_heads"], case["width"], case["page"]
    q, c = _lengths(case["queries"]), _lengths(case["contexts"])
    n, tokens = len(q), sum(q)
    per = [(x + page - 1) // page for x in c]
    pages = sum(per) + 3
    order = torch.randperm(pages, generator=gen, device=_DEV).to(torch.int32)
    at = torch.tensor([sum(per[:b]) for b in range(n)], device=_DEV)
    slot = torch.arange(max(per), device=_DEV)
    used = slot[None, :] < torch.tensor(per, device=_DEV)[:, None]
    table = torch.where(used, order[(at[:, None] + slot).clamp(max=pages - 1)], -1).to(torch.int32)
    pool = (pages, kv_heads, page, width)
    key = normal(*pool).to(torch.bfloat16)
    value = None if case["latent"] else normal(*pool).to(torch.bfloat16)
    key_scale = value_scale = None
    if case["dtype"] == "e4m3":
        key, key_scale = _quantised(key.float())
        if value is not None:
            value, value_scale = _quantised(value.float())
    s = {
        "op": case["op"], "heads": heads, "kv_heads": kv_heads, "width": width, "page": page,
        "tokens": tokens, "longest": max(q), "max_len": max(c), "latent": case["latent"],
        "key": key, "value": value, "key_scale": key_scale, "value_scale": value_scale,
        "table": table.contiguous(),
        "start": torch.tensor([sum(q[:b]) for b in range(n + 1)], device=_DEV, dtype=torch.int32),
        "length": torch.tensor(c, device=_DEV, dtype=torch.int32),
    }
    if case["op"] == "append":
        # the projection of the step: q, k and v heads of a token side by side (a latent alone)
        out_heads = 0 if case["latent"] else heads
        sides = 1 if case["latent"] else 2
        s["q_heads"] = out_heads
        s["qkv"] = normal(tokens, (out_heads + sides * kv_heads) * width).to(torch.bfloat16)
        if not case["latent"]:
            exponent = torch.arange(0, width, 2, device=_DEV, dtype=torch.float64) / width
            angle = torch.arange(max(4096, max(c)), device=_DEV, dtype=torch.float64)[:, None] * 10000.0 ** -exponent
            s["rope"] = (angle.cos().float(), angle.sin().float())
        else:
            s["rope"] = None
    elif case["op"] == "attend":
        s["q"] = normal(tokens, heads, width).to(torch.bfloat16)
        s["window"], s["sinks"] = case["window"], case["sinks"]
        s["scale"] = (96 if case["latent"] else width) ** -0.5
    return s


# ------------------------------------------------------------------------------------ own calls
def _run_own(s):
    b = _bridge()
    if s["op"] == "sample":
        return b.b200_sample(s["logits"], s["uniform"], temperature=s["temperature"],
                             top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    kv = b.PagedKV(s["key"], s["value"], s["key_scale"], s["value_scale"])
    if s["op"] == "read":
        return _some(b.b200_paged_gather(kv, s["table"], s["length"], s["max_len"]))
    if s["op"] == "attend":
        return b.b200_paged_attention(s["q"], kv, s["table"], s["start"], s["length"],
                                      window=s["window"], sinks=s["sinks"], scale=s["scale"])
    q = b.b200_paged_append(kv, s["qkv"], s["table"], s["start"], s["length"], s["q_heads"],
                            rope=s["rope"])
    if s["key_scale"] is None:
        return _some([q, s["key"], s["value"]])
    return _some([q, *b.b200_paged_gather(kv, s["table"], s["length"], s["max_len"])])


def _some(values):
    return [v for v in values if v is not None]


# ----------------------------------------------------------------------------------- plain form
def _token_places(s):
    """(sequence, index in its chunk, position) of every row of the batch."""
    start, i = s["start"].long(), torch.arange(s["tokens"], device=_DEV)
    seq = torch.searchsorted(start[1:], i, right=True)
    own_len = start[1:] - start[:-1]
    index = i - start[seq]
    return seq, index, s["length"].long()[seq] - own_len[seq] + index


def _dense(s, pool, scale, dtype):
    """A pool's rows as [sequences, kv heads, longest context, width], rows past a context zero."""
    p = torch.arange(s["max_len"], device=_DEV)
    page = s["table"].long()[:, p // s["page"]].clamp(min=0)
    rows = pool.view(torch.uint8)[page, :, p % s["page"]].view(pool.dtype) if pool.dtype == _E4M3 \
        else pool[page, :, p % s["page"]]
    x = _values(rows, None if scale is None else scale[page, :, p % s["page"]], dtype)
    inside = p[None, :] < s["length"].long()[:, None]
    return torch.where(inside[:, :, None, None], x, 0).transpose(1, 2)


def _rotated(x, cos, sin):
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack([even * cos - odd * sin, even * sin + odd * cos], -1).flatten(-2)


def _plain_append(s):
    seq, _, pos = _token_places(s)
    heads, kvh, width = s["q_heads"], s["kv_heads"], s["width"]
    x = s["qkv"].float().view(s["tokens"], -1, width)
    q, k, v = x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:]
    if s["rope"] is not None:
        cos, sin = (t[pos][:, None] for t in s["rope"])
        q, k = _rotated(q, cos, sin), _rotated(k, cos, sin)
    page, row = s["table"].long()[seq, pos // s["page"]], pos % s["page"]
    for pool, scale, new in ((s["key"], s["key_scale"], k), (s["value"], s["value_scale"], v)):
        if pool is None:
            continue
        if scale is None:
            pool[page, :, row] = new.to(torch.bfloat16)
        else:
            numbers, byte = _quantised(new)
            pool.view(torch.uint8)[page, :, row] = numbers.view(torch.uint8)
            scale[page, :, row] = byte
    q = q.to(torch.bfloat16) if heads else None
    if s["key_scale"] is None:
        return _some([q, s["key"], s["value"]])
    return _some([q, *_plain_read(s)])


def _plain_read(s):
    out = [_dense(s, s["key"], s["key_scale"], torch.float32).to(torch.bfloat16).contiguous()]
    if s["value"] is not None:
        out.append(_dense(s, s["value"], s["value_scale"], torch.float32).to(torch.bfloat16).contiguous())
    return out


def _plain_attend(s):
    seq, index, pos = _token_places(s)
    n, kvh, group = s["length"].numel(), s["kv_heads"], s["heads"] // s["kv_heads"]
    longest, keys = s["longest"], s["max_len"]
    q = torch.zeros(n, longest, s["heads"], s["width"], device=_DEV)
    q[seq, index] = s["q"].float()
    at = torch.full((n, longest), -1, device=_DEV, dtype=torch.long)
    at[seq, index] = pos
    j = torch.arange(keys, device=_DEV)
    seen = j <= at[:, :, None]
    if s["window"]:
        seen &= (j > at[:, :, None] - s["window"]) | (j < s["sinks"])
    k = _dense(s, s["key"], s["key_scale"], torch.float32)
    v = k if s["value"] is None else _dense(s, s["value"], s["value_scale"], torch.float32)
    q = q.view(n, longest, kvh, group, s["width"]).permute(0, 2, 3, 1, 4).reshape(n, kvh, group * longest, -1)
    score = (q @ k.transpose(-1, -2)).view(n, kvh, group, longest, keys).mul_(s["scale"])
    score.masked_fill_(~seen[:, None, None], _NEG)
    score = torch.exp_(score.sub_(score.amax(-1, keepdim=True).clamp(min=-3e38)))
    total = score.sum(-1, keepdim=True)
    out = score.view(n, kvh, group * longest, keys) @ v
    out = out.view(n, kvh, group, longest, -1) / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4).reshape(n, longest, s["heads"], -1)[seq, index].to(torch.bfloat16)


def _plain_sample(s):
    """In 64 bits: a draw next to a border between two tokens has to fall on the right side."""
    logits, vocab = s["logits"].double(), s["logits"].shape[1]
    t = s["temperature"].double()[:, None]
    greedy = t == 0
    x, index = torch.sort(logits / torch.where(greedy, 1.0, t), dim=1, descending=True, stable=True)
    w = torch.exp(x - x[:, :1])
    rank = torch.arange(vocab, device=_DEV)[None, :]
    k = s["top_k"].long()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0)
    before = w.cumsum(1) - w
    p, all_p = s["top_p"].double()[:, None], (s["top_p"] >= 1)[:, None]
    keep = (all_p | (before < p * w.sum(1, keepdim=True))) & (w >= s["min_p"].double()[:, None])
    keep &= ~greedy
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, 0))
    cdf = kept.cumsum(1)
    total = cdf[:, -1:]
    token = (cdf > s["uniform"].double()[:, None] * total).long().argmax(1, keepdim=True)
    return token, torch.log(kept.gather(1, token) / total)[:, 0].float()


@torch.no_grad()
def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend,
            "sample": _plain_sample}[state["op"]](state)


# ------------------------------------------------------------------------------------------ work
def work(case):
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a subtraction, an exponential and a sum for each token
        return {"bytes": 2 * rows * vocab + 20 * rows + 12 * rows, "flops": 3 * rows * vocab}
    q, c = _lengths(case["queries"]), _lengths(case["contexts"])
    kvh, width, heads = case["kv_heads"], case["width"], case["heads"]
    sides = 1 if case["latent"] else 2
    row = kvh * sides * (2 * width if case["dtype"] == "bf16" else width + 1)  # of one token
    lists = 4 * (2 * len(c) + 1) + sum(4 * -(-x // case["page"]) for x in c)
    dense = 2 * kvh * sides * width * max(c) * len(c)
    if case["op"] == "read":
        return {"bytes": row * sum(c) + dense + lists, "flops": kvh * sides * width * sum(c)}
    if case["op"] == "append":
        q_heads = 0 if case["latent"] else heads
        b = 2 * sum(q) * (q_heads + kvh * sides) * width + 2 * sum(q) * q_heads * width + row * sum(q) + lists
        b += 0 if case["latent"] else 4 * width * len({p for x, y in zip(q, c) for p in range(y - x, y)})
        if case["dtype"] == "e4m3":
            b += row * sum(c) + dense
        return {"bytes": b, "flops": 3 * sum(q) * (q_heads + kvh) * width}
    window, sinks = case["window"] or 1 << 40, case["sinks"]
    pairs = rows = 0
    for x, y in zip(q, c):
        first = y - x
        lo = max(0, first - window + 1)  # the first key that the chunk's first token still has in its window
        rows += y - lo + min(sinks, lo)
        ramp = max(0, min(y, window) - first)  # tokens whose window reaches back to the start
        pairs += ramp * first + ramp * (ramp + 1) // 2
        late = range(first + ramp, y)
        if late:
            extra = [min(sinks, p - window + 1) for p in (late[0], late[-1])]
            pairs += len(late) * window
            pairs += len(late) * sinks if extra[0] == sinks else sum(min(sinks, p - window + 1) for p in late)
    return {"bytes": row * rows + 4 * sum(q) * heads * width + lists, "flops": 4 * pairs * heads * width}


# ------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """The definition in 64 bits, one sequence (or one row of logits) after the other."""
    s = prepare(case, seed)
    if s["op"] == "sample":
        return _exact_sample(s)
    length = s["length"].tolist()
    if s["op"] == "append":
        _exact_write(s)
    if s["op"] == "read" or (s["op"] == "append" and s["key_scale"] is not None):
        dense = []
        for pool, scale in ((s["key"], s["key_scale"]), (s["value"], s["value_scale"])):
            if pool is not None:
                out = torch.zeros(len(length), s["kv_heads"], s["max_len"], s["width"], device=_DEV, dtype=torch.float64)
                for b, n in enumerate(length):
                    out[b, :, :n] = _exact_rows(s, pool, scale, b, n)
                dense.append(out)
        return dense if s["op"] == "read" else _some([s["exact_q"], *dense])
    if s["op"] == "append":
        return _some([s["exact_q"], s["exact_key"], s["exact_value"]])
    start, group = s["start"].tolist(), s["heads"] // s["kv_heads"]
    out = torch.zeros(s["tokens"], s["heads"], s["width"], device=_DEV, dtype=torch.float64)
    for b, n in enumerate(length):
        first, last = start[b], start[b + 1]
        k = _exact_rows(s, s["key"], s["key_scale"], b, n)
        v = k if s["value"] is None else _exact_rows(s, s["value"], s["value_scale"], b, n)
        for lo in range(first, last, 512):
            hi = min(last, lo + 512)
            p = torch.arange(n - last + lo, n - last + hi, device=_DEV)[:, None]
            j = torch.arange(n, device=_DEV)[None, :]
            hidden = j > p
            if s["window"]:
                hidden = hidden | ((p - j >= s["window"]) & (j >= s["sinks"]))
            for h in range(s["heads"]):
                z = s["q"][lo:hi, h].double() @ k[h // group].T * s["scale"]
                z[hidden] = _NEG
                out[lo:hi, h] = torch.softmax(z, 1) @ v[h // group]
    return out


def _exact_rows(s, pool, scale, b, n):
    """[kv heads, n, width] of sequence b in 64 bits."""
    pages = s["table"][b, : -(-n // s["page"])].long()
    x = pool[pages] if pool.dtype != _E4M3 else pool.view(torch.uint8)[pages].view(_E4M3)
    x = x.double()
    if scale is not None:
        x = x * torch.exp2(scale[pages].double() - 127)[..., None]
    return x.transpose(0, 1).reshape(s["kv_heads"], -1, s["width"])[:, :n]


def _exact_write(s):
    heads, kvh, width, page = s["q_heads"], s["kv_heads"], s["width"], s["page"]
    start, length = s["start"].tolist(), s["length"].tolist()
    x = s["qkv"].double().view(s["tokens"], -1, width).clone()
    places = torch.cat([torch.arange(n - (start[b + 1] - start[b]), n, device=_DEV) for b, n in enumerate(length)])
    if s["rope"] is not None:
        turn = torch.complex(s["rope"][0][places].double(), s["rope"][1][places].double())[:, None]
        spun = torch.view_as_complex(x[:, :heads + kvh].reshape(s["tokens"], heads + kvh, width // 2, 2)) * turn
        x[:, :heads + kvh] = torch.view_as_real(spun).flatten(-2)
    s["exact_q"] = x[:, :heads] if heads else None
    wide = {"key": s["key"], "value": s["value"]}
    if s["key_scale"] is None:
        wide = {n: None if p is None else p.double() for n, p in wide.items()}
    for side, new in (("key", x[:, heads:heads + kvh]), ("value", x[:, heads + kvh:])):
        if wide[side] is None:
            continue
        for b, n in enumerate(length):
            lo, hi = start[b], start[b + 1]
            p = torch.arange(n - (hi - lo), n, device=_DEV)
            at, row = s["table"][b].long()[p // page], p % page
            if s["key_scale"] is None:
                wide[side][at, :, row] = new[lo:hi]
            else:
                numbers, byte = _quantised(new[lo:hi])
                wide[side].view(torch.uint8)[at, :, row] = numbers.view(torch.uint8)
                s[side + "_scale"][at, :, row] = byte
    s["exact_key"], s["exact_value"] = wide["key"], wide["value"]


def _exact_sample(s):
    tokens, logs = [], []
    for r in range(s["logits"].shape[0]):
        x = s["logits"][r].double()
        t, k = float(s["temperature"][r]), int(s["top_k"][r])
        if t == 0:
            tokens.append(int(torch.nonzero(x == x.max())[0]))
            logs.append(0.0)
            continue
        w = torch.exp((x - x.max()) / t)
        order = torch.argsort(x, descending=True, stable=True)
        if 0 < k < x.numel():
            order = order[:k]
        top_p, mass = float(s["top_p"][r]), w[order]
        if top_p < 1:
            taken = torch.cat([mass.new_zeros(1), mass.cumsum(0)[:-1]]) < top_p * mass.sum()
            taken[0] = True
            order = order[taken]
        order = torch.cat([order[:1], order[1:][w[order[1:]] >= float(s["min_p"][r])]])
        kept = torch.zeros_like(w)
        kept[order] = w[order]
        cdf = kept.cumsum(0)
        token = int(torch.searchsorted(cdf, float(s["uniform"][r]) * float(cdf[-1]), right=True).clamp(max=x.numel() - 1))
        tokens.append(token)
        logs.append(math.log(float(kept[token]) / float(cdf[-1])) if float(kept[token]) > 0 else _NEG)
    return torch.tensor(tokens, device=_DEV)[:, None], torch.tensor(logs, device=_DEV, dtype=torch.float64)
