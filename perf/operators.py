"""Workloads of the bounded-cache attention operators: attention with a window and sink tokens (forward, and a
training step with its gradients), attention of new tokens over a paged key/value cache, and eviction from a
cache by accumulated attention weight.

`run` computes a case with elementary torch operations in 32 bits, or, where `own` is true, through
byteir_amd.ops; `exact` evaluates the definitions in 64 bits, one sequence and head at a time."""
import math

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    sink = dict(op="sink_fwd", wr=0, layout="bshd")
    train = dict(op="sink_train", wr=0, layout="bshd")
    paged = dict(op="paged", sq=1, wl=-1, sinks=0, new=1, weights=False)
    evict = dict(op="evict", short=0)
    return [
        # a short prompt of one user: launch latency counts
        dict(sink, name="sink_prompt_short", dtype="fp16", b=1, sq=300, sk=300, h=8, hk=8, d=64, wl=127, sinks=4),
        # a long prompt, grouped heads, the usual four sinks
        dict(sink, name="sink_prompt_long", dtype="bf16", b=1, sq=8192, sk=8192, h=32, hk=8, d=128, wl=1023, sinks=4),
        # a prompt's next chunk against what is cached, an odd head dimension, heads outermost in memory
        dict(sink, name="sink_chunk", dtype="fp16", b=2, sq=1000, sk=9001, h=16, hk=16, d=80, wl=2047, sinks=64, layout="bhsd"),
        # fine-tuning on short ragged-length sequences
        dict(train, name="train_small", dtype="fp16", b=2, sq=777, sk=777, h=16, hk=16, d=64, wl=255, sinks=1),
        # long-context training of one sequence
        dict(train, name="train_long", dtype="bf16", b=1, sq=8192, sk=8192, h=32, hk=8, d=128, wl=2047, sinks=4),
        # many sinks (a shared instruction prefix), few key/value heads, a head dimension between the powers of two
        dict(train, name="train_prefix", dtype="bf16", b=2, sq=2048, sk=2048, h=16, hk=2, d=96, wl=511, sinks=128),
        # one chat, just begun: latency
        dict(paged, name="paged_one_short", dtype="fp16", b=1, short=300, long=300, h=32, hk=8, d=128, page=16),
        # a full serving batch of unequal lengths
        dict(paged, name="paged_batch", dtype="bf16", b=64, short=1000, long=8191, h=32, hk=8, d=128, page=64),
        # long streams served with a window and sinks
        dict(paged, name="paged_window", dtype="bf16", b=8, short=60001, long=65500, h=32, hk=8, d=128, page=128, wl=4095, sinks=4),
        # four drafted tokens a sequence, weights accumulated for a later eviction
        dict(paged, name="paged_weights", dtype="fp16", b=8, sq=4, short=9000, long=16380, h=16, hk=16, d=64, page=32, new=4, weights=True),
        # one prompt's cache cut to a quarter
        dict(evict, name="evict_one", dtype="fp16", b=1, short=4096, long=4096, hk=8, d=128, budget=1024, sinks=4, recent=256, page=16),
        # a batch of long prompts, unequal lengths
        dict(evict, name="evict_batch", dtype="bf16", b=16, short=5001, long=16384, hk=8, d=128, budget=4096, sinks=4, recent=1024, page=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["sink_fwd", "sink_train", "paged", "paged", "evict"])
    dtype = rng.choice(["fp16", "bf16"])
    hk = rng.choice([1, 2, 3, 4, 8, 16])
    h = hk * rng.choice([1, 1, 2, 3, 4, 8])
    d = rng.choice([32, 64, 64, 128, 128, 40, 72, 80, 96, 160, 192, 256])
    if op in ("sink_fwd", "sink_train"):
        train = op == "sink_train"
        b = _log(rng, 1, 4)
        while True:  # within the largest listed cases
            sq = _log(rng, 32 if train else 1, 8192)
            sk = sq if train or rng.random() < 0.5 else min(16384, sq + _log(rng, 1, 8192))
            if b * h * sq * sk * max(d, 64) <= 32 * 8192 * 8192 * 128 // 4:
                break
        wl = _log(rng, 16, 4096)
        return dict(op=op, dtype=dtype, b=b, sq=sq, sk=sk, h=h, hk=hk, d=d, wl=wl, wr=0 if rng.random() < 0.8 else _log(rng, 1, 64),
                    sinks=rng.choice([0, 1, 4, 4, 4, 16, 33, 64, 100, 200]), layout=rng.choice(["bshd", "bshd", "bhsd"]))
    b = _log(rng, 1, 64)
    if op == "paged":
        while True:
            long = _log(rng, 1, 65536)
            if b * long * hk * d <= 64 * 8192 * 8 * 128 // 2:
                break
        short = rng.randint(max(1, long // 4), long)
        sq = rng.choice([1, 1, 1, 2, 4, 7])
        windowed = rng.random() < 0.4
        return dict(op=op, dtype=dtype, b=b, sq=sq, short=short, long=long, h=h, hk=hk, d=d, page=rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 256]),
                    wl=_log(rng, 1, 8192) if windowed else -1, sinks=rng.choice([1, 4, 4, 40]) if windowed else 0,
                    new=sq if rng.random() < 0.7 else 0, weights=rng.random() < 0.4)
    while True:
        long = _log(rng, 2, 65536)
        if b * long * hk * d <= 16 * 16384 * 8 * 128:
            break
    short = rng.randint(max(1, long // 4), long)
    budget = max(1, int(long * rng.uniform(0.1, 0.9)))
    recent = int(budget * rng.choice([0.0, 0.25, 0.5]))
    sinks = min(rng.choice([0, 1, 4]), budget - recent)
    return dict(op=op, dtype=dtype, b=b, short=short, long=long, hk=hk, d=d, budget=budget, sinks=sinks, recent=recent, page=rng.choice([1, 16, 32, 64, 100]))


def _lengths(c):
    """The lengths of a batch: evenly from short to long, the longest first (prepare shuffles their order)."""
    b = c["b"]
    return [c["long"] - (c["long"] - c["short"]) * i // max(1, b - 1) for i in range(b)]


def _cap(c):  # pages that a sequence's table names, with one to spare
    return (c["long"] + c.get("new", 0) + c["page"] - 1) // c["page"] + 1


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, b, d, hk = _DT[c["dtype"]], c["b"], c["d"], c["hk"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dt)

    s = {"case": c, "scale": 1.0 / math.sqrt(d)}
    if c["op"] in ("sink_fwd", "sink_train"):
        def rows(n, heads):
            return normal(b, n, heads, d) if c["layout"] == "bshd" else normal(b, heads, n, d).transpose(1, 2)

        s.update(q=rows(c["sq"], c["h"]), k=rows(c["sk"], hk), v=rows(c["sk"], hk))
        if c["op"] == "sink_train":
            s["do"] = normal(b, c["sq"], c["h"], d)
        return s
    order = torch.randperm(b, generator=g, device="cuda")
    lens = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")[order]
    s["lens"] = lens
    if c["op"] == "paged":
        n, page = _cap(c), c["page"]
        pages = b * n + 3
        s.update(q=normal(b, c["sq"], c["h"], d), k_pages=normal(pages, page, hk, d), v_pages=normal(pages, page, hk, d),
                 table=torch.randperm(pages, generator=g, device="cuda")[: b * n].to(torch.int32).view(b, n).contiguous(),
                 k_new=None, v_new=None, weights=None, weights_out=None)
        if c["new"]:
            s.update(k_new=normal(b, c["new"], hk, d), v_new=normal(b, c["new"], hk, d))
        if c["weights"]:
            s["weights"] = torch.rand(b, hk, n * page, generator=g, device="cuda")
            s["weights_out"] = torch.zeros(b, hk, n * page, device="cuda")
        return s
    long, page = c["long"], c["page"]
    n = (c["budget"] + page - 1) // page
    pages = b * n + 1
    # accumulated weights: a few keys hold most of it, some have never been seen (equal weights of zero)
    w = torch.rand(b, hk, long, generator=g, device="cuda").pow_(8)
    w *= torch.rand(b, hk, long, generator=g, device="cuda") > 0.1
    s.update(k=normal(b, long, hk, d), v=normal(b, long, hk, d), weights=w,
             k_out=torch.zeros(pages, page, hk, d, dtype=dt, device="cuda"), v_out=torch.zeros(pages, page, hk, d, dtype=dt, device="cuda"),
             out_table=torch.randperm(pages, generator=g, device="cuda")[: b * n].to(torch.int32).view(b, n).contiguous(),
             weights_out=torch.zeros(b, hk, n * page, device="cuda"), kept=torch.zeros(b, hk, c["budget"], dtype=torch.int32, device="cuda"),
             lens_out=torch.zeros(b, dtype=torch.int32, device="cuda"))
    return s


def _visible(sq, keys, wl, wr, sinks, device):
    """[.., sq, keys]: which keys each query row sees; `keys` a number, or a [b] tensor of per-sequence lengths
    against its longest."""
    i = torch.arange(sq, device=device)
    if isinstance(keys, tuple):
        keys, width = keys
        sk = keys.view(-1, 1, 1)
    else:
        sk, width = keys, keys
    j = torch.arange(width, device=device)
    at = i[:, None] + (sk - sq)  # the key that the row stands at
    hi = torch.minimum(at + 1 + wr, torch.as_tensor(sk, device=device)) if wr >= 0 else torch.as_tensor(sk, device=device).expand(at.shape)
    vis = j < hi
    if wl >= 0:
        vis = vis & ((j >= at - wl) | (j < sinks))
    return vis


def _heads(t, hk):
    """[b, s, h, d] -> [b, hk, (h / hk) * s, d] in 32 bits."""
    b, s, h, d = t.shape
    return t.float().view(b, s, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, h // hk * s, d)


def _rows(t, s, h, dt):
    """The inverse of _heads, rounded to `dt`."""
    b, hk, n, d = t.shape
    return t.view(b, hk, n // s, s, d).permute(0, 3, 1, 2, 4).reshape(b, s, h, d).to(dt)


def _softmax(x):
    """Row maxima and sums of exp over the last axis, a row of -inf counted as empty -> P, lse, empty."""
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = (x - m).exp_()
    l = e.sum(-1, keepdim=True)
    empty = l == 0
    return e.div_(torch.where(empty, torch.ones_like(l), l)), torch.where(empty, torch.full_like(m, math.inf), m + l.log()).squeeze(-1)


def _sink(s, train):
    c, q, k, v, scale = s["case"], s["q"], s["k"], s["v"], s["scale"]
    b, sq, h, d = q.shape
    hk = k.shape[2]
    if own:
        from byteir_amd import ops
        window = (c["wl"], c["wr"])
        o, lse = ops.flash_attn_sink_fwd(q, k, v, scale, window=window, n_sink=c["sinks"])
        if not train:
            return o, lse
        return (o, lse) + tuple(ops.flash_attn_sink_bwd(s["do"], q, k, v, o, lse, scale, window=window, n_sink=c["sinks"]))
    qf, kf, vf = _heads(q, hk), _heads(k, hk), _heads(v, hk)
    vis = _visible(sq, c["sk"], c["wl"], c["wr"], c["sinks"], q.device).repeat(h // hk, 1)
    x = torch.matmul(qf, kf.transpose(-1, -2)).mul_(scale).masked_fill_(~vis, -math.inf)
    p, lse = _softmax(x)
    o = torch.matmul(p, vf)
    out = _rows(o, sq, h, q.dtype), lse.view(b, h, sq)
    if not train:
        return out
    do = _heads(s["do"], hk)
    ds = torch.matmul(do, vf.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, kf).mul_(scale)
    dk = torch.matmul(ds.transpose(-1, -2), qf).mul_(scale)
    dv = torch.matmul(p.transpose(-1, -2), do)
    return out + (_rows(dq, sq, h, q.dtype), _rows(dk, c["sk"], hk, k.dtype), _rows(dv, c["sk"], hk, v.dtype))


def _paged(s):
    c, q, lens, table = s["case"], s["q"], s["lens"], s["table"]
    kp, vp, w, w_out = s["k_pages"], s["v_pages"], s["weights"], s["weights_out"]
    more = [] if s["k_new"] is None else [kp, vp]  # the cache as the call leaves it
    if own:
        from byteir_amd import ops
        return list(ops.flash_attn_paged(q, kp, vp, table, lens, s["scale"], window=(c["wl"], 0), n_sink=c["sinks"],
                                         k_new=s["k_new"], v_new=s["v_new"], weights=w, weights_out=w_out)) + more
    b, sq, h, d = q.shape
    hk, page = c["hk"], c["page"]
    if c["new"]:
        at = lens.long()[:, None] + torch.arange(c["new"], device=q.device)
        pg = table.long().gather(1, at // page)
        kp[pg, at % page] = s["k_new"]
        vp[pg, at % page] = s["v_new"]
    keys = lens.long() + c["new"]
    kf = kp[table.long()].reshape(b, -1, hk, d).permute(0, 2, 1, 3).float()
    vf = vp[table.long()].reshape(b, -1, hk, d).permute(0, 2, 1, 3).float()
    width = kf.shape[2]
    vis = _visible(sq, (keys, width), c["wl"], 0, c["sinks"], q.device)  # [b, sq, width]
    x = torch.matmul(_heads(q, hk), kf.transpose(-1, -2)).mul_(s["scale"]).masked_fill_(~vis.repeat(1, h // hk, 1)[:, None], -math.inf)
    p, lse = _softmax(x)
    out = [_rows(torch.matmul(p, vf), sq, h, q.dtype), lse.view(b, h, sq)]
    if w is not None:
        j = torch.arange(width, device=q.device)
        total = p.sum(2) + torch.where(j < lens[:, None, None], w, torch.zeros_like(w))
        w_out.copy_(torch.where(j < keys[:, None, None], total, w_out))
        out.append(w_out)
    return out + more


def _evict(s):
    c, w, lens = s["case"], s["weights"], s["lens"]
    budget, page = c["budget"], c["page"]
    if own:
        from byteir_amd import ops
        ops.flash_attn_evict(s["k"], s["v"], w, lens, budget, n_sink=c["sinks"], n_recent=c["recent"], k_out=s["k_out"], v_out=s["v_out"],
                             out_table=s["out_table"], weights_out=s["weights_out"], seqlens_out=s["lens_out"], kept=s["kept"])
        return s["kept"], s["k_out"], s["v_out"], s["weights_out"], s["lens_out"]
    b, hk, long = w.shape
    d = c["d"]
    j = torch.arange(long, device=w.device)
    n = lens.long().clamp(max=budget)  # rows kept of each sequence
    ln = lens.long()[:, None, None]
    rank = torch.where((j < c["sinks"]) | (j >= ln - c["recent"]), torch.full_like(w, math.inf), w)
    rank = torch.where(j < ln, rank, torch.full_like(w, -math.inf))
    best = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    i = torch.arange(budget, device=w.device)
    live = i < n[:, None]  # [b, budget]
    best = torch.where(live[:, None], best, torch.full_like(best, long)).sort(-1).values
    kept = torch.where(live[:, None], best, torch.full_like(best, -1)).to(torch.int32)
    src = best.clamp(max=long - 1)
    rows = src.permute(0, 2, 1)[..., None].expand(b, budget, hk, d)
    pg = s["out_table"].long()[:, i // page]
    pb, pi = torch.nonzero(live, as_tuple=True)
    s["k_out"][pg[pb, pi], pi % page] = s["k"].gather(1, rows)[pb, pi]
    s["v_out"][pg[pb, pi], pi % page] = s["v"].gather(1, rows)[pb, pi]
    s["weights_out"][:, :, :budget] = torch.where(live[:, None], w.gather(2, src), s["weights_out"][:, :, :budget])
    s["lens_out"].copy_(n)
    s["kept"].copy_(kept)
    return s["kept"], s["k_out"], s["v_out"], s["weights_out"], s["lens_out"]


def run(s):
    op = s["case"]["op"]
    if op == "paged":
        return _paged(s)
    if op == "evict":
        return _evict(s)
    return _sink(s, op == "sink_train")


def _pairs(sq, sk, wl, wr, sinks):
    """(query, key) pairs that are visible."""
    n = 0
    for i in range(sq):
        at = i + sk - sq
        hi = max(0, min(sk, at + 1 + wr)) if wr >= 0 else sk
        lo = min(hi, max(0, at - wl)) if wl >= 0 else 0
        n += hi - lo + min(lo, sinks)
    return n


def work(c):
    b, d, hk = c["b"], c["d"], c["hk"]
    if c["op"] in ("sink_fwd", "sink_train"):
        pairs = b * c["h"] * _pairs(c["sq"], c["sk"], c["wl"], c["wr"], c["sinks"])
        qs, ks, stat = b * c["sq"] * c["h"] * d * 2, b * c["sk"] * hk * d * 2, b * c["h"] * c["sq"] * 4
        if c["op"] == "sink_fwd":  # q, k, v read; o, lse written
            return {"bytes": 2 * qs + 2 * ks + stat, "flops": 4 * d * pairs}
        return {"bytes": 4 * qs + 4 * ks + stat, "flops": 14 * d * pairs}  # q, k, v, do read; o, lse, dq, dk, dv written
    if c["op"] == "paged":
        rows = flops = 0
        for n in _lengths(c):
            keys = n + c["new"]
            seen = min(keys, c["wl"] + c["sq"] + c["sinks"]) if c["wl"] >= 0 else keys
            rows += seen
            flops += 4 * d * c["h"] * _pairs(c["sq"], keys, c["wl"], 0, c["sinks"])
        moved = rows * hk * d * 4 + 2 * b * c["sq"] * c["h"] * d * 2 + b * c["new"] * hk * d * 4
        return {"bytes": moved + (sum(_lengths(c)) * hk * 8 if c["weights"] else 0), "flops": flops}
    kept = sum(min(n, c["budget"]) for n in _lengths(c))
    return {"bytes": sum(_lengths(c)) * hk * 4 + kept * hk * (d * 8 + 8), "flops": 0}


def _attend64(q, k, v, vis, scale, do=None):
    """One key/value head in 64 bits: q [n, d] (the rows of its query heads), k, v [sk, d], vis [n, sk]."""
    x = (q @ k.T) * scale
    x[~vis] = -math.inf
    lse = torch.logsumexp(x, -1)
    none = lse == -math.inf
    p = torch.exp(x - torch.where(none, torch.zeros_like(lse), lse)[:, None])
    o = p @ v
    lse[none] = math.inf
    if do is None:
        return o, lse, p
    ds = p * (do @ v.T - (do * o).sum(-1, keepdim=True))
    return o, lse, scale * (ds @ k), scale * (ds.T @ q), p.T @ do


def exact(c, seed):
    s = prepare(c, seed)
    hk = c["hk"]
    if c["op"] == "evict":
        return None  # nothing is computed: rows are chosen and moved
    q = s["q"]
    b, sq, h, d = q.shape
    g = h // hk
    if c["op"] in ("sink_fwd", "sink_train"):
        train = c["op"] == "sink_train"
        o, lse = torch.empty(b, sq, h, d, dtype=torch.float64, device=q.device), torch.empty(b, h, sq, dtype=torch.float64, device=q.device)
        dq = torch.empty_like(o)
        dk, dv = torch.empty(b, c["sk"], hk, d, dtype=torch.float64, device=q.device), torch.empty(b, c["sk"], hk, d, dtype=torch.float64, device=q.device)
        at = torch.arange(sq, device=q.device)[:, None] + c["sk"] - sq
        j = torch.arange(c["sk"], device=q.device)
        vis = ((j >= at - c["wl"]) | (j < c["sinks"])) & (j <= at + c["wr"])
        for i in range(b):
            for head in range(h):
                kv = head // g
                r = _attend64(q[i, :, head].double(), s["k"][i, :, kv].double(), s["v"][i, :, kv].double(), vis, s["scale"],
                              s["do"][i, :, head].double() if train else None)
                o[i, :, head], lse[i, head] = r[0], r[1]
                if train:
                    dq[i, :, head] = r[2]
                    if head % g:
                        dk[i, :, kv] += r[3]
                        dv[i, :, kv] += r[4]
                    else:
                        dk[i, :, kv], dv[i, :, kv] = r[3], r[4]
        return (o, lse, dq, dk, dv) if train else (o, lse)
    o, lse = torch.empty(b, sq, h, d, dtype=torch.float64, device=q.device), torch.empty(b, h, sq, dtype=torch.float64, device=q.device)
    w = s["weights_out"].double() if c["weights"] else None
    for i in range(b):
        n = int(s["lens"][i])
        pages = s["table"][i].long()
        k, v = s["k_pages"][pages].flatten(0, 1)[:n], s["v_pages"][pages].flatten(0, 1)[:n]
        if c["new"]:
            k, v = torch.cat([k, s["k_new"][i]]), torch.cat([v, s["v_new"][i]])
        m = n + c["new"]
        at = torch.arange(sq, device=q.device)[:, None] + m - sq
        j = torch.arange(m, device=q.device)
        vis = (((j >= at - c["wl"]) | (j < c["sinks"])) if c["wl"] >= 0 else j >= 0) & (j <= at)
        for head in range(hk):
            r = _attend64(q[i, :, head * g:(head + 1) * g].transpose(0, 1).reshape(g * sq, d).double(), k[:, head].double(), v[:, head].double(),
                          vis.repeat(g, 1), s["scale"])
            o[i, :, head * g:(head + 1) * g] = r[0].view(g, sq, d).transpose(0, 1)
            lse[i, head * g:(head + 1) * g] = r[1].view(g, sq)
            if w is not None:
                w[i, head, :m] = r[2].sum(0)
                w[i, head, :n] += s["weights"][i, head, :n].double()
    out = [o, lse] + ([w] if w is not None else [])
    return out + ([None, None] if c["new"] else [])
