"""Plain 64-bit forms of the paged key-value cache functions, sequence by sequence on the CPU, and builders of pools."""
import math

import torch

FORMATS = (None, "mxint8", "mxfp8_e4m3", "mxfp8_e5m2", "mxfp4")
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative
_SPEC = {"mxfp8_e4m3": (4, 3), "mxfp8_e5m2": (5, 2), "mxfp4": (2, 1)}


def minifloat(code: int, e: int, f: int) -> float:
    exp, man = code >> f & ((1 << e) - 1), code & ((1 << f) - 1)
    bias = (1 << (e - 1)) - 1
    mag = man * 2.0 ** (1 - bias - f) if exp == 0 else (1 + man / (1 << f)) * 2.0 ** (exp - bias)
    return -mag if code >> (e + f) & 1 else mag


def values(codes, scales, fmt):
    """float64 [..., head_dim] of rows of codes and scale bytes [..., head_dim / 32]"""
    if fmt is None:
        return codes.double()
    if fmt == "mxint8":
        x, bias = codes.double(), 134
    else:
        e, f = _SPEC[fmt]
        if fmt == "mxfp4":
            codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
        tab = torch.tensor([minifloat(c, e, f) for c in range(1 << (1 + e + f))], dtype=torch.float64)
        x, bias = tab[codes.long()], 127
    s = torch.exp2(scales.double() - bias)
    s[scales == 255] = math.nan
    return x * s.repeat_interleave(32, -1)


class Pool:
    """pages with random contents for sequences of the given lengths; what no sequence reaches is poisoned (NaN rows,
    NaN scales), and so is the memory around the pages where ``strided``"""

    def __init__(self, gen, lengths, heads, dim, page, fmt, dtype, extra_slots=0, spare=2, strided=False, scale_lo=120, scale_hi=130):
        b = len(lengths)
        self.fmt, self.dtype, self.page, self.dim, self.heads, self.lengths = fmt, dtype, page, dim, heads, list(lengths)
        self.max_length = max(lengths) + extra_slots
        n_tab = max(1, -(-self.max_length // page))
        n = b * n_tab + spare
        self.table = torch.randperm(n, generator=gen)[: b * n_tab].view(b, n_tab).to(torch.int32)
        width = dim // 2 if fmt == "mxfp4" else dim
        shape = (n, heads, page, width)
        self.ks = self.vs = None
        if fmt is None:
            self.k, self.v = (torch.randn(shape, generator=gen).to(dtype) for _ in range(2))
        else:
            if fmt == "mxint8":
                self.k, self.v = (torch.randint(-128, 128, shape, generator=gen).to(torch.int8) for _ in range(2))
                mid = 0
            else:
                self.k, self.v = (torch.randint(0, 256, shape, generator=gen).to(torch.uint8) for _ in range(2))
                if fmt == "mxfp8_e4m3":  # the codes that the packed formats reserve are never written
                    for t in (self.k, self.v):
                        t[(t & 127) == 127] -= 1
                elif fmt == "mxfp8_e5m2":
                    for t in (self.k, self.v):
                        t[(t & 124) == 124] -= 8
                mid = {"mxfp8_e4m3": -6, "mxfp8_e5m2": -13, "mxfp4": 0}[fmt]
            self.ks = torch.randint(scale_lo + mid, scale_hi + mid, (n, heads, page, dim // 32), generator=gen).to(torch.uint8)
            self.vs = torch.randint(scale_lo + mid, scale_hi + mid, (n, heads, dim // 32, page), generator=gen).to(torch.uint8)
        live = torch.zeros(n, page, dtype=torch.bool)
        for i, m in enumerate(lengths):
            for t in range(m):
                live[int(self.table[i, t // page]), t % page] = True
        self.live = live
        dead = ~live
        if fmt is None:
            self.k.transpose(1, 2)[dead] = math.nan
            self.v.transpose(1, 2)[dead] = math.nan
        else:
            self.ks.transpose(1, 2)[dead] = 255
            self.vs.permute(0, 3, 1, 2)[dead] = 255
        self.strided = strided

    def to(self, dev):
        """keyword arguments of the functions, on the device"""
        k, v = self.k, self.v
        if self.strided:  # [pages, page, heads, 1.5 rows] memory seen as [pages, heads, page, row]
            def spread(t):
                n, h, p, w = t.shape
                extra = max(32 // t.element_size(), w // 2)
                big = torch.empty((n, p, h, w + extra), dtype=t.dtype, device=dev)
                big.fill_(math.nan if t.dtype.is_floating_point else 127)
                view = big[..., :w].permute(0, 2, 1, 3)
                view.copy_(t)
                return view
            k, v = spread(k), spread(v)
        else:
            k, v = k.to(dev), v.to(dev)
        kw = dict(k_pages=k, v_pages=v, page_table=self.table.to(dev))
        if self.fmt is not None:
            kw.update(kv_format=self.fmt, k_scales=self.ks.to(dev), v_scales=self.vs.to(dev))
        return kw

    def rows(self, b, n, k=None, v=None, ks=None, vs=None):
        """float64 keys and values [heads, n, dim] of sequence b"""
        k, v = (self.k if k is None else k), (self.v if v is None else v)
        ks, vs = (self.ks if ks is None else ks), (self.vs if vs is None else vs)
        t = torch.arange(n)
        page, at = self.table[b, t // self.page].long(), t % self.page
        sk = sv = None
        if self.fmt is not None:
            sk, sv = ks[page, :, at].transpose(0, 1), vs[page, :, :, at].transpose(0, 1)
        return values(k[page, :, at].transpose(0, 1), sk, self.fmt), values(v[page, :, at].transpose(0, 1), sv, self.fmt)


def attend(q, k, v, scaling, mask, dtype):
    """one sequence: q [heads, dim], k, v [kv_heads, n, dim] float64, mask [n] or None.
    Returns out, probabilities [heads, n], and how far the kernel's out and probabilities may be off."""
    heads, dim = q.shape
    kvh, n, _ = k.shape
    out, tol_o = torch.zeros(heads, dim, dtype=torch.float64), torch.zeros(heads, dim, dtype=torch.float64)
    probs, tol_p = torch.zeros(heads, n, dtype=torch.float64), torch.zeros(heads, n, dtype=torch.float64)
    keep = torch.ones(n, dtype=torch.bool) if mask is None else mask > -math.inf
    if not bool(keep.any()):
        return out, probs, tol_o, tol_p
    half = HALF[torch.float32]
    for h in range(heads):
        kk, vv = k[h // (heads // kvh)][keep], v[h // (heads // kvh)][keep]
        add = 0.0 if mask is None else mask[keep].double()
        prod = q[h].double() * kk
        x = prod.sum(-1) * scaling + add
        e = torch.exp(x - x.max())
        p = e / e.sum()
        out[h], probs[h, keep] = p @ vv, p
        # fp32: a dot product of dim exact products is off by at most dim half-steps of the sum of magnitudes (any order),
        # scaling and mask round once each; the exponent (x - m) log2e rounds twice and the exponential once or so; the
        # sum of n positive terms and the division add (n / 128 + 16) half-steps (n / 128 terms a lane, then trees)
        dx = (dim + 2) * half * float(prod.abs().sum(-1).max()) * abs(scaling)
        if bool((x > -1e30).any()):
            dx += 2 * half * float(x[x > -1e30].abs().max())
        if dtype == torch.float16:  # a code's value below 2^-14 is widened to within half a step of 2^-24
            dx += abs(scaling) * float(q[h].double().abs().sum()) * 2.0 ** -25
        span = float((x.max() - x).clamp(max=120).max())
        rel = 2 * (dx + 4 * half * span) + (n / 128 + 24) * half
        tol_p[h, keep] = p * rel + 2.0 ** -120
        # a probability enters the product with the values as a number of dtype and the rest as another: what is left out is
        # at most HALF of the rest, which is at most HALF of it (fp16: held 2^11 up, bits below 2^-24 there are lost, half a
        # step of 2^-25 2^-11 each); the result rounds to dtype (fp16 below 2^-14: half a step is 2^-25, once for the result
        # and at most once, the probabilities adding up to 1, for code values widened to fp16); the sums over 2 n products
        # run in fp32
        mass = p @ vv.abs()
        tiny = n * 2.0 ** -36 * vv.abs().amax(0) + 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -126
        tol_o[h] = HALF[dtype] * out[h].abs() + mass * (HALF[dtype] ** 2 + rel + (n / 16 + 24) * half) * (1 + HALF[dtype]) + tiny
    return out, probs, tol_o, tol_p


def evict(pos, w, n, keep, recent, first):
    """source slot of each slot after an eviction, for one row"""
    if n <= keep:
        return list(range(n))
    newest = max(pos[:n])

    def rank(s):  # protected ones, then by weight, NaN last, ties to the lowest slot
        if pos[s] < first or pos[s] > newest - recent:
            return (0, 0.0, s)
        return (1, -w[s], s) if w[s] == w[s] else (2, 0.0, s)

    order = sorted(range(n), key=rank)
    kept = sorted(order[:keep])
    inside = set(s for s in kept if s < keep)
    behind = [s for s in kept if s >= keep]
    src, j = [], 0
    for s in range(keep):
        if s in inside:
            src.append(s)
        else:
            src.append(behind[j])
            j += 1
    return src
