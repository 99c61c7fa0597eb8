"""The paged 8-bit KV cache operators on their own: what each is measured on.

Two operators of a serving step over a cache of pages, each page held in 8-bit integers with one
float32 scale for each (page, key/value head):

  append      the new tokens' keys (position rotation applied on the way) and values into their
              pages; a page's scale grows with its largest value, and the tokens that it already
              holds are brought to the new scale. The queries are rotated in the same call. What
              the touched pages then stand for is read back through the same module (gather).
  attention   attention of each sequence's newest tokens over its pages: causal, optionally limited
              to a sliding window and a few first tokens that stay visible (sinks).

Sequences are ragged: rows cu[s] .. cu[s + 1] - 1 of q, k and v are sequence s's new tokens, at
positions start[s] and on; table[s] lists its pages, -1 where there is none yet.

`run` is the plain form, elementary torch operations in 32 bits; with `own` set it makes the calls a
user makes of uwc_b200.paged.
"""
import math
import os
import random
import sys

import torch

own = False
D = 128                      # head dimension
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "useful-work-coin_b200")
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
PLAIN_SCORES = 32 * 8192 * 8192     # the largest listed case's scores in the plain form
PLAIN_KEYS = 32 * 8192 * 8          # the largest listed case's key rows in the plain form
APPEND_HEADS = 8 * 2048 * 32        # the largest listed append's token heads


def _case(name, op, dtype, S, new, length, H, Hkv, ps, ragged=False, window=0, sinks=0):
    c = dict(op=op, dtype=dtype, S=S, new=new, len=length, ragged=ragged, H=H, Hkv=Hkv, ps=ps, window=window,
             sinks=sinks)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one sequence into its last page: a single user's decode step, latency only
        _case("append token x1", "append", "bf16", 1, 1, 2048, 16, 8, 64),
        # a decode step of a batch, pages filled to different heights (16 query heads per 4 of kv)
        _case("append token x64", "append", "bf16", 64, 1, 8192, 32, 8, 64, ragged=True),
        # eight prompts of 2048 tokens written from position 0
        _case("append prompt 8x2048", "append", "bf16", 8, 2048, 2048, 16, 8, 64),
        # odd chunks of prompts behind what is cached, small pages, fp16
        _case("append chunks", "append", "f16", 13, 777, 3001, 12, 4, 16, ragged=True),
        # one user's first tokens: the smallest attention
        _case("token x1 short", "attention", "bf16", 1, 1, 203, 16, 8, 64),
        # a decode batch of 32 with lengths up to 8192
        _case("token x32 ragged", "attention", "bf16", 32, 1, 8192, 32, 8, 64, ragged=True),
        # one long context: few rows, all the work along the cache
        _case("token x1 long", "attention", "bf16", 1, 1, 131071, 32, 8, 128),
        # a decode batch that sees the last 1024 tokens and the first 4
        _case("token x64 window", "attention", "bf16", 64, 1, 8192, 32, 8, 64, ragged=True, window=1024, sinks=4),
        # four drafted tokens checked for each of 16 sequences
        _case("drafts 16x4", "attention", "f16", 16, 4, 3001, 32, 8, 32, ragged=True),
        # prompts attending to themselves
        _case("prompt 8x2048", "attention", "bf16", 8, 2048, 2048, 16, 8, 64),
        # a long prompt with a sliding window and sinks
        _case("prompt 8192 window", "attention", "bf16", 1, 8192, 8192, 32, 8, 64, window=2048, sinks=4),
        # prompt chunks behind a long cached context, small pages, fp16
        _case("chunks 4x512 of 12289", "attention", "f16", 4, 512, 12289, 32, 8, 16, ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    while True:
        op = rng.choice(("append", "attention", "attention"))
        Hkv, G = rng.choice((1, 2, 4, 8, 8)), rng.choice((1, 2, 3, 4, 4, 7, 8))
        S = _log(rng, 1, 64)
        new = rng.choice((1, 1, _log(rng, 2, 16), _log(rng, 17, 8192)))
        length = max(new, _log(rng, 1, 131072))
        window = rng.choice((0, 0, _log(rng, 64, 4096)))
        sinks = rng.choice((0, 1, 4, 130)) if window else 0
        c = _case(None, op, rng.choice(("bf16", "f16")), S, new, length, Hkv * G, Hkv, rng.choice((16, 32, 64, 128)),
                  ragged=rng.random() < 0.7, window=window if op == "attention" else 0,
                  sinks=sinks if op == "attention" else 0)
        if op == "append":
            fits = S * new * Hkv * (G + 2) <= APPEND_HEADS and S * length * Hkv <= PLAIN_KEYS
        else:
            # over 256 new tokens the padded scores decide, else the gathered keys
            fits = S * new * Hkv * G * length <= PLAIN_SCORES and S * length * Hkv <= PLAIN_KEYS
        if fits:
            return c


def _shape(c):
    """Lengths after the append and new tokens, per sequence: a function of the case alone."""
    r = random.Random("%(S)d %(new)d %(len)d %(ps)d" % c)
    lens, new = [], []
    for i in range(c["S"]):
        full = i == 0 or not c["ragged"]
        lens.append(c["len"] if full else max(1, int(c["len"] * r.uniform(0.02, 1.0))))
        new.append(min(lens[-1], c["new"] if full else max(1, int(c["new"] * r.uniform(0.1, 1.0)))))
    return lens, new


def _cu(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 13)
    dt = TYPES[c["dtype"]]
    S, H, Hkv, ps = c["S"], c["H"], c["Hkv"], c["ps"]
    lens, new = _shape(c)
    start = [n - m for n, m in zip(lens, new)]
    need = [-(-n // ps) for n in lens]
    pages = sum(need) + 3
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    # pages of a pool that has been in use: each sequence's lie anywhere in it
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    width = max(need)
    col = torch.arange(width, device=dev)[None, :]
    first = i32(_cu(need)[:-1])[:, None]
    table = torch.where(col < i32(need)[:, None], order[(first + col).clamp(max=pages - 1).long()], -1).to(torch.int32)
    N = sum(new)
    rows = torch.randn(N, (H + 2 * Hkv) * D, device=dev, generator=g)
    rows *= 0.25 + 1.5 * torch.rand(N, 1, device=dev, generator=g)
    # keys have a few dimensions of much larger values, as trained models' do
    rows.view(N, -1, D)[:, H:H + Hkv, 3::41] *= 4.0
    rows = rows.to(dt)
    q = rows[:, :H * D].view(N, H, D)
    k = rows[:, H * D:(H + Hkv) * D].view(N, Hkv, D)
    v = rows[:, (H + Hkv) * D:].view(N, Hkv, D)

    def held():
        x = torch.empty(pages, Hkv, ps, D, dtype=torch.int8, device=dev)
        for p0 in range(0, pages, 512):
            n = min(512, pages - p0)
            x[p0:p0 + n] = (torch.randn(n, Hkv, ps, D, device=dev, generator=g) * 32).round().clamp(-127, 127)
        return x, 0.01 + 0.03 * torch.rand(pages, Hkv, device=dev, generator=g)
    (kc, sk), (vc, sv) = held(), held()
    st = dict(c=c, q=q, k=k, v=v, cache=dict(k=kc, v=vc, sk=sk, sv=sv), table=table, start=i32(start), cu=i32(_cu(new)),
              max_new=max(new), max_len=max(lens), scale=1.0 / math.sqrt(D))
    if c["op"] == "append":
        pos = torch.arange(c["len"], device=dev, dtype=torch.float64)[:, None]
        inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D))
        ang = torch.cat([pos * inv, pos * inv], 1)
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        back = [s % ps + n for s, n in zip(start, new)]      # from the first touched page's first token on
        st["first"], st["back_cu"], st["back"] = i32([s - s % ps for s in start]), i32(_cu(back)), sum(back)
        st["max_back"] = max(back)
    return st


def run(state):
    c = state["c"]
    if own:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        from uwc_b200 import paged
        if c["op"] == "append":
            q = paged.append(state["k"], state["v"], state["cache"], state["table"], state["start"], state["cu"],
                             state["max_new"], state["cos"], state["sin"], q=state["q"])
            k, v = paged.gather(state["cache"], state["table"], state["first"], state["back_cu"], state["back"],
                                state["max_back"], dtype=TYPES[c["dtype"]])
            return dict(q=q, k=k, v=v)
        return paged.attention(state["q"], state["cache"], state["table"], state["start"], state["cu"],
                               state["max_new"], state["max_len"], scale=state["scale"],
                               window=c["window"] or None, sinks=c["sinks"])
    return _plain_append(state) if c["op"] == "append" else _plain_attention(state)


def _rows_at(first, cu, n):
    """The sequence and the position of each of n ragged rows."""
    i = torch.arange(n, device=cu.device)
    seq = torch.searchsorted(cu, i.to(torch.int32), right=True) - 1
    return seq, (first[seq] + i - cu[seq]).long()


def _plain_append(st):
    cache, table, start, cu = st["cache"], st["table"].long(), st["start"], st["cu"]
    ps, N = st["c"]["ps"], st["q"].shape[0]
    seq, pos = _rows_at(start, cu, N)
    cos, sin = st["cos"][pos][:, None, :], st["sin"][pos][:, None, :]

    def rotated(x):
        x = x.float()
        return x * cos + torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1) * sin

    page, off = table[seq, pos // ps], pos % ps
    # the pages that new tokens land in: one row of them per sequence, the last repeated
    end = start + cu[1:] - cu[:-1]
    most = (st["max_new"] + ps - 2) // ps + 1
    j = (start // ps)[:, None] + torch.arange(most, device=cu.device)[None, :]
    j = torch.minimum(j, ((end - 1) // ps)[:, None]).long()
    ids = table.gather(1, j)
    held = (j[..., None] * ps + torch.arange(ps, device=cu.device)) < start[:, None, None]       # old tokens of a page
    full = torch.full((), 127.0, device=cu.device)

    def put(x, data, scale):
        amax = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1) / full, "amax")
        old = torch.where((j * ps < start[:, None])[..., None], scale[ids], 0.0)
        grown = torch.maximum(old, amax[ids])
        # no old token has a value where the grown scale is 0
        by = torch.where(grown > 0, grown, 1.0)[..., None, None]
        d = data[ids].float()
        again = ((d * old[..., None, None]) / by).round().clamp(-127, 127)
        data[ids] = torch.where(held[:, :, None, :, None], again, d).to(torch.int8)
        scale[ids] = grown
        s = scale[page][..., None]
        qv = torch.where(s > 0, x / torch.where(s > 0, s, 1.0), 0.0).round().clamp(-127, 127)
        data[page[:, None], torch.arange(x.shape[1], device=x.device), off[:, None]] = qv.to(torch.int8)

    put(rotated(st["k"]), cache["k"], cache["sk"])
    put(st["v"].float(), cache["v"], cache["sv"])
    bseq, bpos = _rows_at(st["first"], st["back_cu"], st["back"])
    bpage, boff = table[bseq, bpos // ps], bpos % ps
    heads = torch.arange(st["k"].shape[1], device=cu.device)
    back = lambda d, s: (d[bpage[:, None], heads, boff[:, None]].float() * s[bpage][..., None]).to(st["q"].dtype)  # noqa: E731
    return dict(q=rotated(st["q"]).to(st["q"].dtype), k=back(cache["k"], cache["sk"]), v=back(cache["v"], cache["sv"]))


def _plain_attention(st):
    c, cache, start, cu = st["c"], st["cache"], st["start"], st["cu"]
    S, H, Hkv, ps, T = c["S"], c["H"], c["Hkv"], c["ps"], st["max_new"]
    G, N, dev = H // Hkv, st["q"].shape[0], cu.device
    ids = st["table"].clamp(min=0).long()
    L = ids.shape[1] * ps
    dense = lambda d, s: (d[ids].float() * s[ids][..., None, None]).transpose(1, 2).reshape(S, Hkv, L, D)  # noqa: E731
    t = torch.arange(T, device=dev)
    at = (cu[:-1, None] + t).clamp(max=N - 1).long()
    q = st["q"].float()[at].view(S, T, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hkv, T * G, D)
    s = torch.matmul(q, dense(cache["k"], cache["sk"]).transpose(2, 3)) * st["scale"]
    pos, j = (start[:, None] + t)[..., None], torch.arange(L, device=dev)
    seen = j <= pos
    if c["window"]:
        seen = seen & ((j > pos - c["window"]) | (j < c["sinks"]))
    s = s.view(S, Hkv, T, G, L).masked_fill_(~seen[:, None, :, None, :], float("-inf"))
    p = (s - s.amax(-1, keepdim=True)).exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, Hkv, T * G, L), dense(cache["v"], cache["sv"]))
    seq, pos = _rows_at(start, cu, N)
    o = o.view(S, Hkv, T, G, D)[seq, :, pos - start[seq].long()]
    return o.reshape(N, H, D).to(st["q"].dtype)


def work(case):
    c = case
    lens, new = _shape(c)
    N, H, Hkv, ps = sum(new), c["H"], c["Hkv"], c["ps"]
    if c["op"] == "append":
        start = [n - m for n, m in zip(lens, new)]
        held = sum(s % ps for s in start)                      # old tokens in touched pages
        tables = 2 * D * 4 * len({p for s, n in zip(start, new) for p in range(s, s + n)})
        rows = N * D * 2 * (2 * H + 2 * Hkv)                   # q in and out, k and v in
        cached = 2 * Hkv * D * (N + held)                      # written by the append, read back
        return {"bytes": rows + tables + cached + 2 * cached, "flops": 6.0 * N * D * (H + Hkv)}
    pairs = keys = 0
    for n, m in zip(lens, new):
        w, k = c["window"] or n, c["sinks"]
        # key j is seen from position p when p - w < j <= p or j < k
        def prefix(x):                                          # sum over p in [0, x) of min(p + 1, w) + min(max(p + 1 - w, 0), k)
            a = min(x, w)
            b = max(0, x - w)
            d = min(b, k)
            return a * (a + 1) // 2 + b * w + d * (d + 1) // 2 + (b - d) * k
        pairs += prefix(n) - prefix(n - m)
        lo = max(0, n - m - w + 1)                              # first key in any new token's window
        keys += n - lo + min(lo, k)
    return {"bytes": N * H * D * 2 * 2 + keys * Hkv * 2 * D, "flops": 4.0 * D * H * pairs}


def exact(case, seed):
    st = prepare(case, seed)
    lens, new = _shape(case)
    H, Hkv, ps = case["H"], case["Hkv"], case["ps"]
    table, cache = st["table"].cpu().tolist(), st["cache"]
    if case["op"] == "append":
        return _exact_append(st, lens, new, Hkv, ps, table, cache)
    outs, row = [], 0
    for i, (n, m) in enumerate(zip(lens, new)):
        ids = torch.tensor(table[i][:-(-n // ps)], device="cuda")
        pos = torch.arange(n - m, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None, :]
        hidden = j > pos
        if case["window"]:
            hidden |= (j <= pos - case["window"]) & (j >= case["sinks"])
        o = torch.empty(m, H, D, dtype=torch.float64, device="cuda")
        for h in range(Hkv):
            K = (cache["k"][ids, h].double() * cache["sk"][ids, h].double()[:, None, None]).reshape(-1, D)[:n]
            V = (cache["v"][ids, h].double() * cache["sv"][ids, h].double()[:, None, None]).reshape(-1, D)[:n]
            for a in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                x = st["q"][row:row + m, a].double() @ K.T
                x.mul_(1.0 / math.sqrt(D)).masked_fill_(hidden, -math.inf)
                o[:, a] = torch.softmax(x, 1) @ V
        outs.append(o)
        row += m
    return torch.cat(outs)


def _exact_append(st, lens, new, Hkv, ps, table, cache):
    cos, sin = st["cos"].double(), st["sin"].double()
    qs, ks, vs, row = [], [], [], 0

    def turn(x, p):
        lo, hi = x[..., :D // 2], x[..., D // 2:]
        a, b = cos[p, None], sin[p, None]
        return torch.cat([lo * a[..., :D // 2] - hi * b[..., :D // 2], hi * a[..., D // 2:] + lo * b[..., D // 2:]], -1)

    for i, (n, m) in enumerate(zip(lens, new)):
        p = torch.arange(n - m, n, device="cuda")
        take = lambda t: t[row:row + m].double()  # noqa: E731
        qs.append(turn(take(st["q"]), p))
        for x, data, scale, into in ((turn(take(st["k"]), p), cache["k"], cache["sk"], ks),
                                     (take(st["v"]), cache["v"], cache["sv"], vs)):
            base = (n - m) // ps * ps
            held = n - m - base                                 # old tokens of the first page
            total = -(-(n - base) // ps) * ps
            old_page = table[i][base // ps]
            # what the touched pages hold before any rounding, the old tokens as their 8-bit values
            y = torch.zeros(total, Hkv, D, dtype=torch.float64, device="cuda")
            y[held:n - base] = x
            s = y.abs().amax(-1).view(-1, ps, Hkv).amax(1) / 127.0
            if held:
                s0 = scale[old_page].double()
                y[:held] = data[old_page, :, :held].double().transpose(0, 1) * s0[None, :, None]
                s[0] = torch.maximum(s[0], s0)
            s = s.repeat_interleave(ps, 0)[..., None]
            z = torch.where(s > 0, y / torch.where(s > 0, s, 1.0), 0.0).round().clamp(-127, 127) * s
            into.append(z[:n - base])
        row += m
    return dict(q=torch.cat(qs), k=torch.cat(ks), v=torch.cat(vs))
