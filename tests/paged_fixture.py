"""Ragged paged batches for the tests, and the paged operators' plain forms: attention in 64 bits from
the definition, append in numpy float32 (one IEEE operation a step, as the operator is defined)."""
import math

import numpy as np
import torch

D = 128


class Batch:
    """Sequences of `lens` tokens of which the last `new` are new; lens None: an idle slot with `new` rows.
    Pages are taken from a shuffled pool; the table is filled with -1 past each sequence's last page."""

    def __init__(self, lens, new, ps, seed=0, spare=2, extra_rows=0, width=None):
        r = np.random.default_rng(seed)
        self.ps, self.lens, self.new = ps, lens, new
        self.start = [-1 if n is None else n - m for n, m in zip(lens, new)]
        need = [0 if n is None else -(-n // ps) for n in lens]
        self.pages = max(1, sum(need) + spare)
        order = r.permutation(self.pages)
        self.width = width or max(1, max(need))
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for s, c in enumerate(need):
            self.table[s, :c] = order[at:at + c]
            at += c
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.cu[-1]) + extra_rows
        self.max_new, self.max_len = max(new), max([n for n in lens if n is not None], default=0)

    def device(self, dev):
        t = lambda x: torch.tensor(np.asarray(x, np.int32), device=dev)
        return t(self.table), t(self.start), t(self.cu)


def random_cache(b: Batch, Hkv, dev, seed=0, spread=1.0):
    """Pages holding values: integers of any size, scales over a factor of 10 ** spread."""
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    i8 = lambda: torch.randint(-127, 128, (b.pages, Hkv, b.ps, D), device=dev, generator=g, dtype=torch.int8)
    sc = lambda: 0.02 * 10 ** (spread * (torch.rand(b.pages, Hkv, device=dev, generator=g) - 0.5))
    return dict(k=i8(), v=i8(), sk=sc(), sv=sc())


def attention64(q, cache, b: Batch, scale, window, sinks):
    """(o, tol part) in float64 on q's device: o from the definition, and for every output value
    sum_j p_j |v_j| and the row's largest sum_d |q_d k_d| scale, which bound the rounding."""
    H, Hkv = q.shape[1], cache["k"].shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    absv, smax = torch.zeros_like(o), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for s, (n, m) in enumerate(zip(b.lens, b.new)):
        if n is None or m == 0:
            continue
        ids = torch.tensor(b.table[s, :-(-n // b.ps)].astype(np.int64), device=q.device)
        dense = lambda d, sc: (d[ids].double() * sc[ids].double()[..., None, None]).transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
        K, V = dense(cache["k"], cache["sk"]), dense(cache["v"], cache["sv"])
        r0 = int(b.cu[s])
        x = q[r0:r0 + m].double().view(m, Hkv, H // Hkv, D)
        pos, j = torch.arange(n - m, n, device=q.device)[:, None], torch.arange(n, device=q.device)[None, :]
        seen = j <= pos
        if window is not None:
            seen &= (j > pos - window) | (j < sinks)
        sc = torch.einsum("mhgd,hnd->mhgn", x, K) * scale
        sc.masked_fill_(~seen[:, None, None, :], -math.inf)
        top = sc.amax(-1, keepdim=True)
        p = torch.exp(sc - torch.where(top.isinf(), 0.0, top))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        o[r0:r0 + m] = torch.einsum("mhgn,hnd->mhgd", p, V).reshape(m, H, D)
        absv[r0:r0 + m] = torch.einsum("mhgn,hnd->mhgd", p, V.abs()).reshape(m, H, D)
        smax[r0:r0 + m] = torch.einsum("mhgd,hnd->mhgn", x.abs(), K.abs()).amax(-1).reshape(m, H) * scale
    return o, absv, smax


def tolerance(o, absv, smax, dtype):
    """What the arithmetic can lose: the output's rounding (the type's unit roundoff, half its eps), the weights'
    rounding to 11 bits, and scores in float32: 128 products added in some order, each addition off by
    2^-24 of the sums of magnitudes (2^-17 of smax in all), twice as the row's maximum enters too."""
    return torch.finfo(dtype).eps / 2 * o.abs() + (2.0 ** -11 + 2.0 ** -16 * smax[..., None]) * absv * 1.01 + 1e-7


def f32(x):
    return np.asarray(x, np.float32)


def turn(x, cos, sin):
    """The rotation, one rounding per operation."""
    rot = np.concatenate([-x[..., D // 2:], x[..., :D // 2]], -1)
    return f32(f32(x * cos) + f32(rot * sin))


def append_plain(k, v, cache, b: Batch, cos, sin):
    """The cache (numpy dict, updated) after appending rows k, v (float32 values)."""
    for s, (n, m) in enumerate(zip(b.lens, b.new)):
        if n is None or m == 0:
            continue
        r0, st = int(b.cu[s]), n - m
        p = np.arange(st, n)
        for x, dn, sn in ((turn(f32(k[r0:r0 + m]), cos[p][:, None], sin[p][:, None]), "k", "sk"),
                          (f32(v[r0:r0 + m]), "v", "sv")):
            for slot in range(st // b.ps, (n - 1) // b.ps + 1):
                base, page = slot * b.ps, b.table[s, slot]
                lo, hi = max(st, base), min(n, base + b.ps)
                y = x[lo - st:hi - st]                                    # (t, Hkv, 128)
                mag = np.where(np.isfinite(y), np.abs(y), f32(0))
                new = f32(mag.max((0, 2)) / f32(127))
                old = cache[sn][page] if lo > base else f32(np.zeros_like(new))
                scale = np.maximum(old, new)
                with np.errstate(all="ignore"):
                    w = np.rint(f32(y / scale[None, :, None]))
                    w = np.where(scale[None, :, None] > 0, np.clip(w, -127, 127), 0)
                    w = np.where(np.isnan(y), 0, w)
                cache[dn][page][:, lo - base:hi - base] = w.transpose(1, 0, 2).astype(np.int8)
                grown = scale > old
                if lo > base and grown.any():
                    h = cache[dn][page][:, :lo - base]
                    again = np.rint(f32(f32(h.astype(np.float32) * old[:, None, None]) / np.where(scale > 0, scale, 1)[:, None, None]))
                    h[grown] = again[grown].astype(np.int8)
                cache[sn][page] = scale
    return cache
