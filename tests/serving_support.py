"""Plain 64-bit statements of the serving operators, and ragged paged batches to run them on."""
from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn
HALF_BF16 = 2.0 ** -8  # half a step of bf16, relative


def scale_exponent(amax: torch.Tensor) -> torch.Tensor:
    """The least e with amax <= 448 * 2**e, clamped to -110 .. 119 (by trial, not by bits)."""
    e = torch.full_like(amax, -110, dtype=torch.int32)
    for t in range(-110, 119):
        e = torch.where(amax.double() > 448.0 * 2.0 ** t, t + 1, e)
    return e


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of fp32 -> (e4m3 numbers, scale bytes): the definition of an 8-bit row."""
    amax = torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf).abs().amax(-1)
    e = scale_exponent(amax)
    scaled = (x.double() * torch.exp2(-e.double())[..., None]).clamp(-448.0, 448.0)
    return scaled.float().to(E4M3), (e + 127).to(torch.uint8)


def dequantise(numbers: torch.Tensor, scale: torch.Tensor | None) -> torch.Tensor:
    x = numbers.double()
    return x if scale is None else x * torch.exp2(scale.double() - 127)[..., None]


def rope_tables(positions: int, dim: int, theta: float = 10000.0):
    exponent = torch.arange(0, dim, 2).double() / dim
    angle = torch.arange(positions).double()[:, None] * theta ** -exponent
    return angle.cos().float(), angle.sin().float()


def rotate_f32(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """(e cos - o sin, e sin + o cos), every product and sum one fp32 rounding."""
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack([e * cos - o * sin, e * sin + o * cos], -1).flatten(-2)


class Paged:
    """A paged cache on the CPU (fp32 values it stands for) and its device copy."""

    def __init__(self, contexts, *, kv_heads, dim, page, e4m3=False, latent=False, seed=0,
                 spare=2, scale=1.0, width=None):
        g = torch.Generator().manual_seed(seed)
        self.contexts, self.page, self.kv_heads, self.dim = list(contexts), page, kv_heads, dim
        per = [-(-c // page) for c in self.contexts]
        self.pages = sum(per) + spare
        order = torch.randperm(self.pages, generator=g)
        width = max([1] + per) if width is None else width
        self.table = torch.full((len(per), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(per):
            self.table[b, :n] = order[at:at + n].int()
            at += n
        shape = (self.pages, kv_heads, page, dim)

        def pool():
            x = torch.randn(shape, generator=g) * scale
            return quantise(x) if e4m3 else (x.to(torch.bfloat16), None)

        self.key, self.key_scale = pool()
        self.value, self.value_scale = (None, None) if latent else pool()

    def rows(self, side: str, b: int, n: int | None = None) -> torch.Tensor:
        """[kv heads, n, dim] in 64 bits: sequence b's rows of the pool ``side``."""
        pool, scale = getattr(self, side), getattr(self, side + "_scale")
        n = self.contexts[b] if n is None else n
        ids = self.table[b, : -(-n // self.page)].long()
        x = dequantise(pool.view(torch.uint8)[ids].view(E4M3) if pool.dtype == E4M3 else pool[ids],
                       None if scale is None else scale[ids])
        return x.transpose(0, 1).reshape(self.kv_heads, -1, self.dim)[:, :n]

    def device(self, device="cuda"):
        from parrot_b200 import bridge

        def to(t):
            return None if t is None else t.to(device)
        return bridge.PagedKV(to(self.key), to(self.value), to(self.key_scale), to(self.value_scale))


def starts(queries) -> torch.Tensor:
    return torch.tensor([sum(queries[:b]) for b in range(len(queries) + 1)], dtype=torch.int32)


def visible(positions: torch.Tensor, keys: int, window: int, sinks: int) -> torch.Tensor:
    p, j = positions[:, None], torch.arange(keys)[None, :]
    seen = j <= p
    if window:
        seen = seen & ((p - j < window) | (j < sinks))
    return seen


def attention(q: torch.Tensor, cache: Paged, queries, window: int, sinks: int, scale: float):
    """(out, bound): the formula in 64 bits, and how far a kernel may be from it.

    The kernels round each p to bf16 before the product with v (half a step,
    relative) and the result once to bf16.  The scores are sums of D exact
    products in fp32 and the exponential is fp32: together they move a p by
    less than 2**-12 for scores up to a few hundred (D + 3 roundings of 2**-24
    of a score's terms).  With A = sum p |v| / sum p that is
    2**-8 (A + |out|) + 2**-12 A, and 2**-16 A for the product of the two roundings.
    """
    heads, group = q.shape[1], q.shape[1] // cache.kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64)
    mass = torch.zeros(q.shape, dtype=torch.float64)
    first = 0
    for b, n in enumerate(queries):
        c = cache.contexts[b]
        if n == 0:
            continue
        k = cache.rows("key", b)
        v = k if cache.value is None else cache.rows("value", b)
        pos = torch.arange(c - n, c)
        seen = visible(pos, c, window, sinks)
        for h in range(heads):
            z = q[first:first + n, h].double() @ k[h // group].T * scale
            z = z.masked_fill(~seen, -math.inf)
            p = torch.softmax(z, 1)
            p = torch.where(seen, p, 0.0)  # a row that sees nothing: zeros
            # a masked place counts for nothing, whatever it holds
            vv = v[h // group]
            if torch.isfinite(vv).all():
                out[first:first + n, h] = p @ vv
                mass[first:first + n, h] = p @ vv.abs()
            else:
                for i in range(n):
                    out[first + i, h] = p[i][seen[i]] @ vv[seen[i]]
                    mass[first + i, h] = p[i][seen[i]] @ vv[seen[i]].abs()
        first += n
    bound = HALF_BF16 * (mass + out.abs()) + (2.0 ** -12 + 2.0 ** -16) * mass + 1e-30
    return out, bound


def sample_row(logits, u, temperature, top_k, top_p, min_p):
    """(token, log-probability) of one row, in 64 bits."""
    x = logits.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    if float(x.max()) == -math.inf:
        return -1, -math.inf
    best = int(torch.nonzero(x == x.max())[0])
    if not temperature > 0:
        return best, 0.0
    w = torch.where(x == x.max(), 1.0, torch.exp((x - x.max()) / temperature))
    order = [int(i) for i in torch.argsort(-x, stable=True) if x[i] > -math.inf]
    if 0 < top_k < x.numel():
        order = order[:top_k]
    if top_p < 1:
        share, before, kept = top_p * math.fsum(float(w[i]) for i in order), 0.0, []
        for i in order:
            if kept and not before < share:
                break
            kept.append(i)
            before += float(w[i])
        order = kept
    order = order[:1] + [i for i in order[1:] if float(w[i]) >= min_p]
    total = math.fsum(float(w[i]) for i in order)
    run, token = 0.0, None
    for i in sorted(order):
        run += float(w[i])
        if run > u * total:
            token = i
            break
    if token is None:
        token = max(i for i in order if float(w[i]) > 0)
    return token, math.log(float(w[token]) / total)
