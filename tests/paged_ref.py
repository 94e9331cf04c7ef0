"""Plain 64-bit restatements of the paged-cache operators, and the batches their tests use."""
import math

import torch

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dt):
    """The largest relative error of one rounding to dt."""
    return torch.finfo(dt).eps / 2


def rotation(rows, dim, device):
    """f32 tables [rows, dim / 2] whose two halves of a head turn by the same angle."""
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * torch.arange(dim // 2, dtype=torch.float64) / dim)
    return ang.cos().float().to(device), ang.sin().float().to(device)


def norm_rope(x, weight, eps, cos, sin, positions):
    """The result and, per value, the size of the terms it is a sum of (for tolerances)."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    size = y.abs()
    if cos is not None:
        h = cos.shape[1]
        c, s = cos.double()[positions.long()][:, None], sin.double()[positions.long()][:, None]
        a, b = y[..., :h], y[..., h:2 * h]
        size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), size[..., 2 * h:]], -1)
        y = torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * h:]], -1)
    return y, size


def norm_rope_tolerance(y, size, dt):
    """The f32 part: a sum of up to 256 squares (at most 16 fused adds in a thread and 4 across
    lanes: 20 roundings, half of that after the square root) and about six more roundings of 2^-24:
    below 2^-19 of the terms; then one rounding to dt (half its smallest subnormal near zero)."""
    e = 2.0 ** -19 * size
    return e + half_step(dt) * (y.abs() + e) + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


class Batch:
    """Sequences of `lengths` positions, the last `new` of them new, in a shuffled pool of pages.
    order: the memory order of the pool's axes (pages, heads, slots) before head_dim."""

    def __init__(self, new, lengths, q_heads, kv_heads, hd, page, dt, seed=0, device="cuda", order=(0, 1, 2), spare=3,
                 table_fill=-1, pool_fill=None, extra_rows=0):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.new, self.len, self.page, self.hd, self.dt = list(new), list(lengths), page, hd, dt
        self.qh, self.kvh, self.n = q_heads, kv_heads, len(new)
        pages = [-(-x // page) for x in lengths]
        total = sum(pages) + spare
        perm = torch.randperm(total, generator=g, device=device).tolist()
        width = max(pages + [1])
        table, at = torch.full((self.n, width), table_fill, dtype=torch.int32), 0
        for i, p in enumerate(pages):
            table[i, :p] = torch.tensor(perm[at:at + p], dtype=torch.int32)
            at += p
        self.table = table.to(device)
        self.q_start = torch.tensor([0] + torch.tensor(self.new, dtype=torch.int64).cumsum(0).tolist() if self.n else [0],
                                    dtype=torch.int32, device=device)
        self.lengths = torch.tensor(self.len, dtype=torch.int32, device=device)
        self.tokens = sum(new)
        self.max_chunk, self.max_length = max(self.new + [0]), max(self.len + [0])
        size = (total, kv_heads, page)
        inverse = [order.index(i) for i in range(3)]

        def pool():
            shape = [size[i] for i in order] + [hd]
            p = torch.randn(shape, generator=g, device=device).to(dt) if pool_fill is None else torch.full(shape, pool_fill, dtype=dt, device=device)
            return p.permute(*inverse, 3)
        self.k_pool, self.v_pool = pool(), pool()
        rows = self.tokens + extra_rows
        self.q = (1.5 * torch.randn(rows, q_heads, hd, generator=g, device=device)).to(dt)
        self.k = torch.randn(rows, kv_heads, hd, generator=g, device=device).to(dt)
        self.v = torch.randn(rows, kv_heads, hd, generator=g, device=device).to(dt)
        self.gate = torch.rand(rows, q_heads, hd, generator=g, device=device).to(dt)

    def sequence(self, i, pool):
        """[heads, length, hd] of sequence i in 64 bits."""
        p = torch.arange(self.len[i], device=pool.device)
        return pool[self.table[i].long()[p // self.page], :, p % self.page].double().transpose(0, 1)

    def put(self, i, pool, values):
        """Write values [heads, length, hd] as sequence i's positions."""
        p = torch.arange(self.len[i], device=pool.device)
        pool[self.table[i].long()[p // self.page], :, p % self.page] = values.transpose(0, 1).to(pool.dtype)


def visible(new, length, window=0, bits=None, self_visible=False, device="cuda"):
    """[new, length] bool: the keys that each new token sees. bits [length] bool or None."""
    key = torch.arange(length, device=device)[None]
    pos = torch.arange(length - new, length, device=device)[:, None]
    ok = key <= pos
    if window:
        ok = ok & (key > pos - window)
    if bits is not None:
        ok = ok & (bits[None, :length] | (key == pos if self_visible else torch.zeros_like(ok)))
    return ok


def attention(b, scale=None, window=0, bits=None, self_visible=False, gate=None):
    """(out, tolerance) [tokens, q_heads, hd] f64. bits [n, >= max length] bool or None.

    Tolerance, u = the half step of the type and A = the mean of |v| under the same weights: the
    probabilities are rounded to the type (u A); the score is a sum of hd f32 products
    (hd 2^-24 of their sizes, in the exponent, once for a key and once for the sum of all) and a few
    roundings of the exponent, whose size in log2 units stays below 2^7 (2^7 2^-24, twice); the
    weighted values are sums of n f32 products (n 2^-24 A); one rounding at the end, with the gate's."""
    hd, group = b.hd, b.qh // b.kvh
    scale = 1 / math.sqrt(hd) if scale is None else scale
    u = half_step(b.dt)
    out = torch.zeros(b.tokens, b.qh, hd, dtype=torch.float64, device=b.q.device)
    tol = torch.zeros_like(out)
    first = 0
    for i, (n, length) in enumerate(zip(b.new, b.len)):
        if not n:
            continue
        k, v = b.sequence(i, b.k_pool), b.sequence(i, b.v_pool)
        see = visible(n, length, window, None if bits is None else bits[i], self_visible, b.q.device)
        for h in range(b.qh):
            q = b.q[first:first + n, h].double()
            kk, vv = k[h // group], v[h // group]
            used = see.any(0)                       # what nobody sees may hold anything
            kk, vv = torch.where(used[:, None], kk, 0.0), torch.where(used[:, None], vv, 0.0)
            s = (q @ kk.T) * scale
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            total = p.sum(1, keepdim=True)
            p = p / torch.where(total > 0, total, 1.0)
            y, size = p @ vv, p @ vv.abs()
            e = 2 * hd * 2.0 ** -24 * abs(scale) * ((q.abs() @ kk.abs().T) * see).amax(1, keepdim=True)
            err = (u + 2 * e + 2 * 2.0 ** -17 + length * 2.0 ** -24) * size
            if gate is not None:
                gg = gate[first:first + n, h].double()
                y, err = y * gg, err * gg.abs()
            out[first:first + n, h] = y
            tol[first:first + n, h] = err + (u + 2.0 ** -23) * (y.abs() + err) + torch.finfo(b.dt).smallest_normal * torch.finfo(b.dt).eps
        first += n
    return out, tol


def words(bits):
    """[n, positions] bool -> int32 words, bit p % 32 of word p // 32."""
    n, m = bits.shape
    w = -(-m // 32)
    full = torch.zeros(n, w * 32, dtype=torch.int64, device=bits.device)
    full[:, :m] = bits.long()
    x = (full.view(n, w, 32) << torch.arange(32, device=bits.device)).sum(2)
    return torch.where(x >= 2 ** 31, x - 2 ** 32, x).to(torch.int32)


def within(got, want, tol):
    """Every value within its tolerance; the worst share of it, for the message."""
    got = got.double()
    assert torch.isfinite(got).all(), "values that are not finite"
    d = (got - want).abs()
    share = (d / tol).max().item() if d.numel() else 0.0
    assert share <= 1.0, f"off by {share:.3g} times the tolerance (error {d.max().item():.3g})"
