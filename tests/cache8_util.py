"""The 8-bit page format and the operators on it, written out in float64 (a block at a time, token by token)."""
import math

import numpy as np
import torch

BLOCK = 16
TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
E_MIN, E_MAX = -40, 40


def exponent(amax: float, dtype) -> int:
    """Smallest e in [E_MIN, E_MAX] with amax <= TOP 2^e."""
    if amax == 0:
        return E_MIN
    if math.isinf(amax):
        return E_MAX
    e = E_MIN
    while e < E_MAX and amax > TOP[dtype] * 2.0 ** e:
        e += 1
    return e


def encode(x, dtype) -> torch.Tensor:
    """float64 values (already divided by the scale) -> the numbers that the codes stand for, to nearest even."""
    x = torch.nan_to_num(torch.as_tensor(x, dtype=torch.float64), nan=0.0, posinf=TOP[dtype], neginf=-TOP[dtype])
    if dtype == torch.int8:
        return torch.round(x).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)      # three bits behind the leading one
    return (torch.round(x / step) * step).clamp(-448, 448)


def half_step(x, e, dtype) -> torch.Tensor:
    """Largest rounding error of the encoding of x (float64) in a block of exponent e, for magnitudes within the range."""
    x = torch.as_tensor(x, dtype=torch.float64).abs()
    if dtype == torch.int8:
        return torch.full_like(x, 2.0 ** (e - 1))
    return torch.maximum(x * 2.0 ** -4, torch.full_like(x, 2.0 ** (e - 10)))           # subnormal codes are 2^-9 apart


def to_codes(numbers, dtype) -> torch.Tensor:
    return torch.as_tensor(numbers, dtype=torch.float32).to(dtype)


class Pools:
    """The pools of one layer on the CPU, with what the codes stand for in float64."""

    def __init__(self, pages, nkv, page_size, d, dtype, seed=0, garbage=True):
        self.pages, self.nkv, self.page_size, self.d, self.dtype = pages, nkv, page_size, d, dtype
        sub = page_size // BLOCK
        g = torch.Generator().manual_seed(seed)
        raw = lambda *shape: torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)  # noqa: E731
        # what is not written may hold any byte (e4m3: NaN codes among them) and any scale
        self.kcache = raw(pages, nkv, page_size, d).view(dtype) if garbage else torch.zeros(pages, nkv, page_size, d, dtype=torch.uint8).view(dtype)
        self.vcache = raw(pages, nkv, sub, d, BLOCK).view(dtype) if garbage else torch.zeros(pages, nkv, sub, d, BLOCK, dtype=torch.uint8).view(dtype)
        self.kscale = torch.full((pages, nkv, sub), float("nan") if garbage else 2.0 ** -40)
        self.vscale = self.kscale.clone()

    def put(self, page, place, k, v, ke=None, ve=None):
        """Tokens place .. of a page from k, v [n, nkv, d] in float64; exponents per (head, block) chosen if not given."""
        n = k.shape[0]
        for b in range(place // BLOCK, (place + n - 1) // BLOCK + 1):
            lo, hi = max(place, b * BLOCK), min(place + n, (b + 1) * BLOCK)
            for h in range(self.nkv):
                for x, cache, scale, fixed in ((k, self.kcache, self.kscale, ke), (v, self.vcache, self.vscale, ve)):
                    part = x[lo - place:hi - place, h]
                    e = exponent(part.abs().max().item(), self.dtype) if fixed is None else fixed
                    scale[page, h, b] = 2.0 ** e
                    codes = to_codes(encode(part * 2.0 ** -e, self.dtype), self.dtype)
                    if cache is self.kcache:
                        cache[page, h, lo:hi] = codes
                    else:
                        cache[page, h, b, :, lo - b * BLOCK:hi - b * BLOCK] = codes.T

    def values(self, page, place, n):
        """(k, v) [n, nkv, d] of tokens place .. of a page, float64."""
        ks, vs = [], []
        for i in range(place, place + n):
            b = i // BLOCK
            ks.append(self.kcache[page, :, i].double() * self.kscale[page, :, b, None].double())
            vs.append(self.vcache[page, :, b, :, i % BLOCK].double() * self.vscale[page, :, b, None].double())
        return torch.stack(ks), torch.stack(vs)

    def value_scales(self, page, place, n):
        """[n, nkv]: the scale of the value block of each token."""
        return torch.stack([self.vscale[page, :, i // BLOCK].double() for i in range(place, place + n)])

    def on(self, dev):
        return [t.to(dev) for t in (self.kcache, self.vcache, self.kscale, self.vscale)]


class Sequences:
    """Sequences of several lengths in 8-bit pages scattered over a pool."""

    def __init__(self, lengths, nkv, d, page_size, dtype, seed=0, value_scale=None, extra_pages=2):
        g = torch.Generator().manual_seed(seed + 1)
        per = [(n + page_size - 1) // page_size for n in lengths]
        total = sum(per) + extra_pages
        self.pools = Pools(total, nkv, page_size, d, dtype, seed)
        perm = torch.randperm(total, generator=g).tolist()
        self.table = torch.full((len(lengths), max(per) + 2), -1, dtype=torch.int32)
        self.k, self.v, self.vs = [], [], []
        for s, n in enumerate(lengths):
            k, v = torch.randn(n, nkv, d, generator=g).double(), torch.randn(n, nkv, d, generator=g).double()
            if value_scale is not None:
                v = v * value_scale(torch.arange(n).double())[:, None, None]
            ks, vs, sc = [], [], []
            for i in range(per[s]):
                page = perm.pop()
                self.table[s, i] = page
                lo, hi = i * page_size, min(n, (i + 1) * page_size)
                self.pools.put(page, 0, k[lo:hi], v[lo:hi])
                a, b = self.pools.values(page, 0, hi - lo)
                ks.append(a); vs.append(b); sc.append(self.pools.value_scales(page, 0, hi - lo))
            self.k.append(torch.cat(ks)); self.v.append(torch.cat(vs)); self.vs.append(torch.cat(sc))


def attention_with_bound(q, k, v, vs, pos, window, scale, weight_rounding, d, sum_rounding=0.0):
    """q [nq, d], k and v [len, nkv, d], vs [len, nkv] the scale of each token's value block, float64: (out [nq, d], bound on the error of a kernel that rounds its weights by
    ``weight_rounding`` relative to themselves - and its sum by ``sum_rounding`` - and its result to bfloat16).

    out = sum p v.  A weight is off by its rounding and by the error e of its score (natural log units): products in 32 bits
    with d + 16 roundings of terms of total size A = scale sum |q k|; queries below 2^-14 of the head's largest lose up to
    2^-25 of it; 2^-20 for exp2 and the rescalings.  The weights are kept as w = p times the scale of their value block over the largest
    such product, in half precision: one below 2^-14 is subnormal and loses up to 2^-25, times the code of its value.  The
    result is rounded by half a step, 2^-8."""
    lo = max(0, pos - window + 1) if window else 0
    group = q.shape[0] // k.shape[1]
    out, bound = [], []
    for h in range(q.shape[0]):
        kk, vv = k[lo:pos + 1, h // group], v[lo:pos + 1, h // group]
        s = kk @ q[h] * scale
        p = torch.softmax(s, 0)
        o = p @ vv
        A = (kk.abs() @ q[h].abs()).max() * scale
        e = (d + 16) * 2.0 ** -24 * A + 2.0 ** -25 * q[h].abs().max() * kk.abs().sum(1).max() * scale + 2.0 ** -20
        spread = p @ vv.abs()
        sc = vs[lo:pos + 1, h // group]
        small = 2.0 ** -25 * (p * sc).max() * (vv.abs() / sc[:, None]).sum(0)
        out.append(o)
        bound.append(2.0 ** -8 * o.abs() + 1.01 * ((weight_rounding + sum_rounding + 2 * e) * spread + small) + 1e-30)
    return torch.stack(out), torch.stack(bound)
