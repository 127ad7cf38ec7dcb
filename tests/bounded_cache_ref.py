"""The definitions of the bounded-cache operators (attention with a window and sinks and its gradient, over a
paged cache, eviction by weight) in 64 bits, with the error that the kernels' roundings can cause,
element by element.

u is half a step of the storage type (torch.finfo(t).eps / 2 relative to the value); the kernels round

* P to the storage type before P V and P^T dO: each term of the sum is off by at most u of its size;
* O, dQ, dK, dV once at the end: u of the value;
* dS to the storage type before dS K and dS^T Q, and D = dO . O is made from the rounded O.

In 32 bits they carry S = q.k (d products: an error of at most (d + 2) 2^-24 sum |q k|, which the
exponential turns into a relative error of P), the exponent's argument (rounded to 2^-24 of its
size), v_exp_f32 / v_log_f32 (2^-23) and the sums over n keys (n 2^-24 relative: the terms are positive)."""
import math

import torch

E32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(sq, sk, window, n_sink, device="cpu"):
    """[sq, sk]: row i stands at key i + sk - sq; right side of the window first, then its left side or the sinks."""
    wl, wr = window
    at = torch.arange(sq, device=device)[:, None] + (sk - sq)
    j = torch.arange(sk, device=device)[None, :]
    vis = torch.ones(sq, sk, dtype=torch.bool, device=device)
    if wr >= 0:
        vis &= j <= at + wr
    if wl >= 0:
        vis &= (j >= at - wl) | (j < n_sink)
    return vis


def head(q, k, v, scale, vis, do=None, u=0.0):
    """One query head: q [n, d], k, v [sk, d], vis [n, sk] -> dict of values and of their error bounds (name + '_tol')."""
    q, k, v = q.double(), k.double(), v.double()
    d, n_keys = q.shape[1], max(1, k.shape[0])
    # what nobody sees must not matter: zeros in its place
    k, v = (torch.where(vis.any(0)[:, None], t, torch.zeros_like(t)) for t in (k, v))
    s = scale * (q @ k.T)
    s_err = (d + 2) * E32 * scale * (q.abs() @ k.abs().T) + 4 * E32 * s.abs()
    s = s.masked_fill(~vis, -math.inf)
    m = s.amax(1, keepdim=True) if k.shape[0] else torch.full((q.shape[0], 1), -math.inf, dtype=torch.float64, device=q.device)
    none = m == -math.inf
    e = torch.exp(s - torch.where(none, torch.zeros_like(m), m))
    l = e.sum(1, keepdim=True)
    p = e / torch.where(none, torch.ones_like(l), l)
    lse = torch.where(none, torch.full_like(m, math.inf), m + torch.log(l)).squeeze(1)
    worst = s_err.masked_fill(~vis, 0).amax(1, keepdim=True) if k.shape[0] else torch.zeros_like(m)  # of a row's scores
    size = torch.where(none, torch.zeros_like(m), s.masked_fill(~vis, 0).abs().amax(1, keepdim=True) if k.shape[0] else torch.zeros_like(m))
    r = 2 * worst + 4 * E32 * size + 8 * E32 + n_keys * E32  # relative error of P before it is rounded
    o, a = p @ v, p @ v.abs()
    res = {"o": o, "lse": lse, "p": p, "p_tol": p * r,
           "o_tol": u * o.abs() + (u + r) * (1 + u) * a + 1e-30,
           "lse_tol": (r + 4 * E32 * lse.abs().unsqueeze(1).nan_to_num(posinf=0)).squeeze(1)}
    if u:  # results below the normal range of the type (fp16) are rounded to its least step
        res["o_tol"] = res["o_tol"] + u * LEAST[u]
    if do is None:
        return res
    do = do.double()
    dp = do @ v.T
    dd = (do * o).sum(1, keepdim=True)
    ds = p * (dp - dd)
    rb = r + 4 * E32 * torch.where(none, torch.zeros_like(m), lse.unsqueeze(1).nan_to_num(posinf=0).abs())  # P again, from the stored lse
    dd_err = (do.abs() * res["o_tol"]).sum(1, keepdim=True) + (d + 2) * E32 * (do.abs() * o.abs()).sum(1, keepdim=True)
    dp_err = (d + 2) * E32 * (do.abs() @ v.abs().T)
    ds_err = p * (dd_err + dp_err) * (1 + rb) + (u + 2 * rb) * ds.abs() + (p * u * LEAST[u] if u else 0)
    n = q.shape[0]
    if u:  # P and dS too are rounded to the least step of the type where they are small
        ds_err, p_err = ds_err + (u * LEAST[u]) * (p > 0), (u + rb) * p + (u * LEAST[u]) * (p > 0)
    else:
        p_err = rb * p
    res.update(dq=scale * (ds @ k), dk=scale * (ds.T @ q), dv=p.T @ do)
    res["dq_tol"] = u * res["dq"].abs() + scale * ((ds_err + n_keys * E32 * ds.abs()) @ k.abs()) * (1 + u) + 1e-30
    res["dk_err"] = scale * ((ds_err + n * E32 * ds.abs()).T @ q.abs()) * (1 + u)  # before the rounding of the sum over the group
    res["dv_err"] = (p_err + n * E32 * p).T @ do.abs() * (1 + u)
    return res


# the least normal number of each type, by its half step: below it a rounding is off by half a step of IT
LEAST = {half_step(torch.float16): 2.0 ** -14, half_step(torch.bfloat16): 2.0 ** -126}


def attention(q, k, v, scale, window, n_sink, do=None):
    """[b, s, h, d] tensors -> dict: o, lse, (dq, dk, dv) in 64 bits and name + '_tol' of each."""
    b, sq, h, d = q.shape
    sk, hk = k.shape[1], k.shape[2]
    u = half_step(q.dtype)
    vis = visible(sq, sk, window, n_sink, q.device)
    z = lambda *s: torch.zeros(s, dtype=torch.float64, device=q.device)
    out = {"o": z(b, sq, h, d), "lse": z(b, h, sq)}
    if do is not None:
        out.update(dq=z(b, sq, h, d), dk=z(b, sk, hk, d), dv=z(b, sk, hk, d))
    out.update({n + "_tol": torch.zeros_like(t) for n, t in list(out.items())})
    for i in range(b):
        for x in range(h):
            y = x // (h // hk)
            r = head(q[i, :, x], k[i, :, y], v[i, :, y], scale, vis, None if do is None else do[i, :, x], u)
            for n in ("o", "o_tol"):
                out[n][i, :, x] = r[n]
            out["lse"][i, x], out["lse_tol"][i, x] = r["lse"], r["lse_tol"]
            if do is not None:
                out["dq"][i, :, x], out["dq_tol"][i, :, x] = r["dq"], r["dq_tol"]
                for n in ("dk", "dv"):
                    out[n][i, :, y] += r[n]
                    out[n + "_tol"][i, :, y] += r[n + "_err"]
    for n in ("dk", "dv") if do is not None else ():
        out[n + "_tol"] += u * out[n].abs() + u * LEAST[u] + (h // hk) * E32 * out[n].abs() + 1e-30
    if do is not None:
        out["dq_tol"] += u * LEAST[u]
    return out


def rows_of(pages, table, b, n):
    """The first n rows of sequence b and which of them exist -> [n, h_k, d], bool [n]."""
    if table is None:
        return pages[b, :n], torch.ones(n, dtype=torch.bool, device=pages.device)
    num, page = pages.shape[:2]
    j = torch.arange(n, device=pages.device)
    pg = table[b].long()[j // page]
    ok = (pg >= 0) & (pg < num)
    return pages[pg.clamp(0, max(0, num - 1)), j % page], ok


def paged(q, k_pages, v_pages, table, lens, scale, window, n_sink, k_new=None, v_new=None, weights=None, weights_out=None):
    """flash_attn_paged's definition: dict of o, lse, k_pages, v_pages, weights and their tolerances; nothing is changed."""
    b, sq, h, d = q.shape
    hk = k_pages.shape[2]
    u, g = half_step(q.dtype), h // hk
    cap = k_pages.shape[1] * (table.shape[1] if table is not None else 1)
    kp, vp = k_pages.clone(), v_pages.clone()
    n_new = k_new.shape[1] if k_new is not None else 0
    z = lambda *s: torch.zeros(s, dtype=torch.float64, device=q.device)
    out = {"o": z(b, sq, h, d), "lse": torch.full((b, h, sq), math.inf, dtype=torch.float64, device=q.device)}
    out.update(o_tol=torch.zeros_like(out["o"]), lse_tol=torch.zeros_like(out["lse"]))
    w = weights_out.double() if weights_out is not None else None
    w_tol = torch.zeros_like(w) if w is not None else None
    for i in range(b):
        old = int(lens[i])
        if old < 0:
            continue
        for t in range(n_new):
            at = old + t
            if at >= cap:
                break
            pg, r = (i, at) if table is None else (int(table[i, at // kp.shape[1]]), at % kp.shape[1])
            if 0 <= pg < kp.shape[0]:
                kp[pg, r], vp[pg, r] = k_new[i, t], v_new[i, t]
        n = min(cap, old + n_new)
        k, ok = rows_of(kp, table, i, n)
        v, _ = rows_of(vp, table, i, n)
        vis = visible(sq, n, window, n_sink, q.device) & ok[None, :]
        for c in range(hk):
            got = torch.zeros(n, dtype=torch.float64, device=q.device)
            tol = torch.zeros_like(got)
            for x in range(c * g, (c + 1) * g):
                r = head(q[i, :, x], k[:, c], v[:, c], scale, vis, None, u)
                for name in ("o", "o_tol"):
                    out[name][i, :, x] = r[name]
                out["lse"][i, x], out["lse_tol"][i, x] = r["lse"], r["lse_tol"]
                got += r["p"].sum(0)
                # P from the stored lse: its error and the rounding of lse * log2(e) and of the argument
                tol += (r["p_tol"] + r["p"] * (r["lse_tol"] + 8 * E32 * (1 + r["lse"].nan_to_num(posinf=0).abs()))[:, None]).sum(0)
            if w is not None:
                before = torch.zeros(n, dtype=torch.float64, device=q.device)
                if weights is not None:
                    before[:min(old, n)] = weights[i, c, :min(old, n)].double()
                w[i, c, :n] = before + got
                w_tol[i, c, :n] = tol + (g * sq + 1) * E32 * (before.abs() + got)
    out.update(k_pages=kp, v_pages=vp, weights=w, weights_tol=w_tol)
    return out


def evict(weights, lens, cap, budget, n_sink, n_recent):
    """flash_attn_evict's choice: kept [b, h_k, budget] (-1 behind the last) and the lengths after it."""
    b, hk, _ = weights.shape
    kept = torch.full((b, hk, budget), -1, dtype=torch.int32)
    new = lens.cpu().clone()
    for i in range(b):
        n = max(0, min(int(lens[i]), cap))
        if int(lens[i]) >= 0:
            new[i] = min(n, budget)
        for c in range(hk):
            if n <= budget:
                kept[i, c, :n] = torch.arange(n, dtype=torch.int32)
                continue
            w = [float(x) for x in weights[i, c, :n].cpu()]
            key = lambda j: (0, -w[j], j) if w[j] == w[j] else (1, 0.0, j)  # NaN behind everything, ties to the lower row
            middle = sorted(range(n_sink, n - n_recent), key=key)[:budget - n_sink - n_recent]
            rows = list(range(n_sink)) + sorted(middle) + list(range(n - n_recent, n))
            kept[i, c] = torch.tensor(rows, dtype=torch.int32)
    return kept, new


def close(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin], want[~fin]), (what, "infinities differ")
    bad = ~((got - want).abs() <= tol) & fin
    if bool(bad.any()):
        x = (got - want).abs()[fin]
        raise AssertionError((what, f"{int(bad.sum())} of {bad.numel()} off, worst {float(x.max()):.3g}, first at {bad.nonzero()[0].tolist()}: "
                              f"{float(got[bad][0]):.6g} for {float(want[bad][0]):.6g} +- {float(tol[bad][0]):.3g}"))
