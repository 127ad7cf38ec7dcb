"""Attention with a window and sinks (forward, gradients), over a paged cache, and eviction, on the GPU against
their definitions in 64 bits (bounded_cache_ref, with its derived tolerances)."""
import math

import pytest
import torch

import bounded_cache_ref as R
from byteir_amd import ops

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float16):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


SINK_CASES = [
    # b, sq, sk, h, h_k, d, window, n_sink
    (1, 1, 1, 1, 1, 32, (0, 0), 0),
    (2, 1, 700, 8, 2, 128, (100, 0), 4),
    (1, 700, 700, 4, 4, 64, (64, 0), 4),
    (1, 1300, 1300, 4, 2, 128, (200, 0), 4),
    (2, 513, 513, 6, 3, 32, (1, 1), 1),
    (1, 333, 2000, 4, 1, 128, (511, 0), 130),
    (1, 640, 100, 2, 2, 64, (30, 0), 4),        # rows without keys
    (1, 500, 500, 3, 3, 72, (99, 0), 33),
    (1, 300, 900, 2, 1, 192, (128, 5), 16),
    (1, 257, 600, 2, 2, 256, (300, -1), 64),
    (1, 400, 400, 4, 2, 160, (-1, 0), 9),
    (1, 5, 3000, 16, 16, 64, (1500, 0), 4),     # few rows, keys split over workgroups
    (1, 0, 50, 2, 2, 64, (9, 0), 4),
    (1, 50, 0, 2, 2, 64, (9, 0), 4),
    (0, 50, 50, 2, 2, 64, (9, 0), 4),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", SINK_CASES)
def test_sink_forward_and_gradients(case, dtype):
    b, sq, sk, h, hk, d, window, ns = case
    g = gen(sq + sk + d)
    q, do = randn(g, b, sq, h, d, dtype=dtype), randn(g, b, sq, h, d, dtype=dtype)
    k, v = randn(g, b, sk, hk, d, dtype=dtype), randn(g, b, sk, hk, d, dtype=dtype)
    scale = 1 / math.sqrt(d)
    o, lse = ops.flash_attn_sink_fwd(q, k, v, scale, window, ns)
    dq, dk, dv = ops.flash_attn_sink_bwd(do, q, k, v, o, lse, scale, window, ns)
    want = R.attention(q, k, v, scale, window, ns, do)
    for name, got in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        R.close(got, want[name], want[name + "_tol"], (name, case))


@pytest.mark.parametrize("d", [64, 128, 96])
def test_sink_gradient_is_the_derivative(d):
    """The gradient of sum(o * w) against central differences of the 64-bit definition along random directions:
    the kernel's gradient, whose error per element is bounded, against a difference whose own is of order eps^2."""
    g = gen(d)
    b, s, h, hk, window, ns, scale = 1, 150, 2, 1, (30, 0), 3, 1 / math.sqrt(d)
    q, do = randn(g, b, s, h, d), randn(g, b, s, h, d)
    k, v = randn(g, b, s, hk, d), randn(g, b, s, hk, d)
    o, lse = ops.flash_attn_sink_fwd(q, k, v, scale, window, ns)
    grads = ops.flash_attn_sink_bwd(do, q, k, v, o, lse, scale, window, ns)
    want = R.attention(q, k, v, scale, window, ns, do)
    vis = R.visible(s, s, window, ns, "cuda")

    def f(q, k, v):
        return sum((R.head(q[0, :, x], k[0, :, 0], v[0, :, 0], scale, vis)["o"] * do[0, :, x].double()).sum() for x in range(h))

    args = [q.double(), k.double(), v.double()]
    for i, name in enumerate(("dq", "dk", "dv")):
        t = torch.randn(args[i].shape, generator=g, device="cuda", dtype=torch.float64)
        eps = 1e-4
        hi, lo = (f(*[a + e * t if j == i else a for j, a in enumerate(args)]) for e in (eps, -eps))
        diff = float((hi - lo) / (2 * eps))
        got = float((grads[i].double() * t).sum())
        tol = float((want[name + "_tol"] * t.abs()).sum()) + 1e-5 * abs(diff)
        assert abs(got - diff) <= tol, (name, got, diff, tol)


def test_sink_layouts():
    """[b, h, s, d] storage, one packed buffer, an expanded (broadcast) key/value pair and its dense gradient."""
    g = gen(3)
    b, s, h, d, window, ns = 2, 300, 4, 64, (70, 0), 4
    packed = randn(g, b, s, 3, h, d)
    q, k, v = packed.unbind(2)
    do = randn(g, b, h, s, d).transpose(1, 2)
    want = R.attention(q, k, v, 0.125, window, ns, do)
    o, lse = ops.flash_attn_sink_fwd(q, k, v, 0.125, window, ns)
    grads = ops.flash_attn_sink_bwd(do, q, k, v, o, lse, 0.125, window, ns)
    for name, got in (("o", o), ("lse", lse), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        R.close(got, want[name], want[name + "_tol"], name)
    k1, v1 = k[:1].expand(b, s, h, d), v[:, :, :1].expand(b, s, h, d)
    want = R.attention(q, k1, v1, 0.125, window, ns, do)
    o, lse = ops.flash_attn_sink_fwd(q, k1, v1, 0.125, window, ns)
    grads = ops.flash_attn_sink_bwd(do, q, k1, v1, o, lse, 0.125, window, ns)
    for name, got in (("o", o), ("lse", lse), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        R.close(got, want[name], want[name + "_tol"], "expanded " + name)


@pytest.mark.parametrize("d", [64, 128, 80])
def test_sink_masked_keys_may_hold_anything(d):
    g = gen(4)
    q, do = randn(g, 1, 60, 4, d), randn(g, 1, 60, 4, d)
    k, v = randn(g, 1, 900, 2, d), randn(g, 1, 900, 2, d)
    k[:, 4:700], v[:, 4:700] = float("nan"), float("inf")
    args = (1 / math.sqrt(d), (140, 0), 4)
    o, lse = ops.flash_attn_sink_fwd(q, k, v, *args)
    grads = ops.flash_attn_sink_bwd(do, q, k, v, o, lse, *args)
    want = R.attention(q, k, v, *args, do)
    for name, got in (("o", o), ("lse", lse), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        R.close(got, want[name], want[name + "_tol"], name)


def test_sink_long_prompt_one_head():
    g = gen(5)
    q, do = randn(g, 1, 6001, 2, 128, dtype=torch.bfloat16), randn(g, 1, 6001, 2, 128, dtype=torch.bfloat16)
    k, v = randn(g, 1, 6001, 1, 128, dtype=torch.bfloat16), randn(g, 1, 6001, 1, 128, dtype=torch.bfloat16)
    args = (128 ** -0.5, (1023, 0), 4)
    o, lse = ops.flash_attn_sink_fwd(q, k, v, *args)
    grads = ops.flash_attn_sink_bwd(do, q, k, v, o, lse, *args)
    want = R.attention(q, k, v, *args, do)
    for name, got in (("o", o), ("lse", lse), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        R.close(got, want[name], want[name + "_tol"], name)


def pages_of(g, b, cap, page, hk, d, dtype, spare=2):
    n = -(-cap // page)
    k, v = randn(g, b * n + spare, page, hk, d, dtype=dtype), randn(g, b * n + spare, page, hk, d, dtype=dtype)
    table = torch.randperm(b * n + spare, generator=g, device="cuda")[:b * n].to(torch.int32).view(b, n).contiguous()
    return k, v, table


PAGED_CASES = [
    # lens, capacity, page, sq, n_new, h, h_k, d, window, n_sink, weights
    ([1], 16, 16, 1, 0, 1, 1, 32, (-1, 0), 0, False),
    ([300, 0, 77, -1], 320, 16, 1, 1, 32, 8, 128, (-1, 0), 0, False),
    ([9000, 31, 4097], 9100, 64, 1, 1, 8, 2, 128, (-1, 0), 0, True),
    ([5000, 2000, 5], 5200, 7, 1, 0, 6, 2, 64, (1000, 0), 4, True),
    ([700, -1, 40], 800, 100, 3, 3, 6, 2, 40, (33, 0), 40, True),
    ([0, 1, 2], 64, 1, 4, 0, 4, 4, 32, (-1, 0), 0, True),
    ([3000, 333], 3100, 24, 40, 40, 8, 1, 96, (-1, 0), 0, True),
    ([250, 100], 256, 32, 70, 70, 2, 1, 256, (50, 2), 3, False),
    ([4000], 4100, 256, 2, 9, 2, 1, 64, (3, 0), 1, True),
    ([1200, 900], 1300, 128, 1, 1, 64, 1, 192, (-1, -1), 0, True),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", PAGED_CASES)
def test_paged(case, dtype):
    lens, cap, page, sq, n_new, h, hk, d, window, ns, weighted = case
    b = len(lens)
    g = gen(cap + page + d)
    k, v, table = pages_of(g, b, cap, page, hk, d, dtype)
    q = randn(g, b, sq, h, d, dtype=dtype)
    kn, vn = (randn(g, b, n_new, hk, d, dtype=dtype), randn(g, b, n_new, hk, d, dtype=dtype)) if n_new else (None, None)
    full = table.shape[1] * page
    w = torch.rand((b, hk, full), generator=g, device="cuda") if weighted else None
    w_out = torch.full((b, hk, full), -7.0, device="cuda") if weighted else None
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    scale = 1 / math.sqrt(d)
    want = R.paged(q, k, v, table, n, scale, window, ns, kn, vn, w, w_out)
    r = ops.flash_attn_paged(q, k, v, table, n, scale, window, ns, kn, vn, w, w_out)
    R.close(r[0], want["o"], want["o_tol"], ("o", case))
    R.close(r[1], want["lse"], want["lse_tol"], ("lse", case))
    assert torch.equal(k, want["k_pages"]) and torch.equal(v, want["v_pages"])
    if weighted:
        R.close(r[2], want["weights"], want["weights_tol"], ("weights", case))


def test_paged_hidden_rows_and_absent_pages():
    g = gen(10)
    k, v, table = pages_of(g, 2, 1600, 16, 2, 64, torch.float16)
    n = torch.tensor([1500, 1450], dtype=torch.int32, device="cuda")
    for at, x in (((0, 3), -1), ((0, 93), k.shape[0]), ((1, 90), 1 << 30), ((1, 0), -(1 << 31)), ((1, 89), -5)):
        table[at] = x
    q = randn(g, 2, 2, 4, 64)
    kn, vn = randn(g, 2, 2, 2, 64), randn(g, 2, 2, 2, 64)
    used = torch.zeros(k.shape[:2], dtype=torch.bool, device="cuda")
    for i in range(2):
        for j in list(range(3)) + list(range(int(n[i]) + 2 - 2 - 600, int(n[i]))):
            if 0 <= int(table[i, j // 16]) < k.shape[0]:
                used[int(table[i, j // 16]), j % 16] = True
    k[~used], v[~used] = float("nan"), float("nan")
    w_out = torch.zeros(2, 2, 1600, device="cuda")
    want = R.paged(q, k, v, table, n, 0.125, (600, 0), 3, kn, vn, None, w_out)
    o, lse, w_out = ops.flash_attn_paged(q, k, v, table, n, 0.125, (600, 0), 3, kn, vn, None, w_out)
    R.close(o, want["o"], want["o_tol"], "o")
    R.close(lse, want["lse"], want["lse_tol"], "lse")
    R.close(w_out, want["weights"], want["weights_tol"], "weights")
    assert torch.equal(k.view(torch.int16), want["k_pages"].view(torch.int16)) and torch.equal(v.view(torch.int16), want["v_pages"].view(torch.int16))


def test_paged_offsets_past_32_bits():
    """A pool of 2^32 elements and more behind its first page: reads, appends and moves at its far end."""
    g = gen(11)
    hk, d, page = 2, 128, 64
    num = (1 << 32) // (page * hk * d) + 40
    k, v = (torch.zeros(num, page, hk, d, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.tensor([[num - 1, 0, num - 7, 1, num - 2], [2, num - 3, num - 4, num - 9, 3]], dtype=torch.int32, device="cuda")
    for p in table.flatten().tolist():
        k[p], v[p] = randn(g, page, hk, d), randn(g, page, hk, d)
    n = torch.tensor([319, 200], dtype=torch.int32, device="cuda")
    q, kn, vn = randn(g, 2, 1, 4, d), randn(g, 2, 1, hk, d), randn(g, 2, 1, hk, d)
    o, lse = ops.flash_attn_paged(q, k, v, table, n, 0.09, k_new=kn, v_new=vn)
    assert torch.equal(k[num - 2, 63], kn[0, 0]) and torch.equal(v[num - 9, 8], vn[1, 0])
    small = table.flatten().long()
    ks, vs = k[small], v[small]
    want = R.paged(q, ks, vs, torch.arange(10, dtype=torch.int32, device="cuda").view(2, 5), n + 1, 0.09, (-1, 0), 0)
    R.close(o, want["o"], want["o_tol"], "o")
    R.close(lse, want["lse"], want["lse_tol"], "lse")
    w = torch.rand(2, hk, 320, generator=g, device="cuda")
    kept, _, _ = ops.flash_attn_evict(k, v, w, n + 1, 100, 2, 10, block_table=table, weights_out=w, seqlens_out=n)
    for i in range(2):
        for c in range(hk):
            src = kept[i, c].long()
            got = k[table[i].long()].flatten(0, 1)[:100, c]
            assert torch.equal(got, ks.view(2, 5, page, hk, d)[i].flatten(0, 1)[src, c])
    assert n.tolist() == [100, 100]


EVICT_CASES = [
    # lens, source rows, budget, n_sink, n_recent, h_k, d, page (0: dense), page of the output
    ([3000, 50, 500, -1], 3000, 500, 4, 100, 8, 64, 16, 32),
    ([100, 97], 100, 96, 0, 0, 1, 128, 0, 7),
    ([40000], 40000, 12000, 1, 1000, 2, 40, 64, 0),
    ([2, 1, 0], 2, 1, 0, 0, 3, 8, 1, 1),
    ([5000, 4999], 5000, 4000, 4000, 0, 2, 128, 128, 128),
    ([900], 800, 700, 2, 3, 1, 256, 50, 50),
]


def rows_equal(new, new_table, old, old_table, i, c, src):
    a, b = R.rows_of(new, new_table, i, len(src))[0][:, c], R.rows_of(old, old_table, i, int(src.max()) + 1 if len(src) else 0)[0][:, c][src]
    return torch.equal(a, b)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", EVICT_CASES)
def test_evict(case, in_place):
    lens, rows, budget, ns, nr, hk, d, page, page_out = case
    b, g = len(lens), gen(case[1])
    dtype = torch.float16 if in_place else torch.bfloat16
    if page:
        k, v, table = pages_of(g, b, rows, page, hk, d, dtype)
        cap = table.shape[1] * page
    else:
        k, v, table, cap = randn(g, b, rows, hk, d, dtype=dtype), randn(g, b, rows, hk, d, dtype=dtype), None, rows
    w = torch.rand((b, hk, cap), generator=g, device="cuda").pow(6)
    w = torch.where(torch.rand((b, hk, cap), generator=g, device="cuda") < 0.3, torch.zeros_like(w), w)
    w[torch.rand((b, hk, cap), generator=g, device="cuda") < 0.02] = float("nan")
    w[torch.rand((b, hk, cap), generator=g, device="cuda") < 0.02] = -0.0
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, n_want = R.evict(w, n, cap, budget, ns, nr)
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    if in_place:
        kept, w_out, n_out = ops.flash_attn_evict(k, v, w, n, budget, ns, nr, block_table=table)
        ko, vo, to = k, v, table
        assert w_out is w and n_out is n
    else:
        to = None
        ko, vo = randn(g, b, budget, hk, d, dtype=dtype), randn(g, b, budget, hk, d, dtype=dtype)
        if page_out:
            ko, vo, to = pages_of(g, b, budget, page_out, hk, d, dtype)
        kept, w_out, n_out = ops.flash_attn_evict(k, v, w, n, budget, ns, nr, table, ko, vo, to)
        assert torch.equal(k, k0) and torch.equal(v, v0)
    assert torch.equal(kept.cpu(), want) and torch.equal(n_out.cpu(), n_want)
    for i in range(b):
        for c in range(hk):
            src = want[i, c][want[i, c] >= 0].long().cuda()
            assert rows_equal(ko, to, k0, table, i, c, src) and rows_equal(vo, to, v0, table, i, c, src)
            assert torch.equal(w_out[i, c, :len(src)].view(torch.int32), w0[i, c, src].view(torch.int32))


def test_streams_workspaces_and_same_bits():
    """Another stream than the current one, scratch of the caller's filled with NaN patterns, two calls at once on two
    streams: always the same bits."""
    g = gen(12)
    q, do = randn(g, 1, 700, 8, 64), randn(g, 1, 700, 8, 64)
    k, v = randn(g, 1, 700, 2, 64), randn(g, 1, 700, 2, 64)
    kp, vp, table = pages_of(g, 2, 3000, 16, 2, 64, torch.float16)
    n, qt = torch.tensor([2900, 150], dtype=torch.int32, device="cuda"), randn(g, 2, 1, 8, 64)

    def run(stream, ws=None):
        o, lse = ops.flash_attn_sink_fwd(q, k, v, 0.125, (100, 0), 4, stream=stream)
        grads = ops.flash_attn_sink_bwd(do, q, k, v, o, lse, 0.125, (100, 0), 4, stream=stream)
        w = torch.empty(2, 2, 3008, device="cuda").fill_(0)
        return (o, lse) + tuple(grads) + tuple(ops.flash_attn_paged(qt, kp, vp, table, n, 0.125, weights_out=w, stream=stream, workspace=ws))

    first = run(None)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    need = ops.flash_attn_workspace_bytes("paged", q.dtype, ops.pack_flash_paged_args(qt, kp, vp, None, None, qt, 0.125, (-1, 0), 0, table.shape[1], 1))
    assert need > 0
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run(s, torch.full((need,), 255, dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(first, r):
            assert torch.equal(a, b)


def test_captured_and_replayed():
    """One graph of the whole run, replayed on new inputs with eager work between, against the eager calls."""
    g = gen(13)
    b, s, h, hk, d, budget = 2, 400, 8, 2, 64, 128
    mk = lambda *shape: torch.zeros(shape, dtype=torch.float16, device="cuda")
    q, k, v, do = mk(b, s, h, d), mk(b, s, hk, d), mk(b, s, hk, d), mk(b, s, h, d)
    kp, vp = mk(40, 16, hk, d), mk(40, 16, hk, d)
    table = torch.arange(24, dtype=torch.int32, device="cuda").view(2, 12) + 3
    lens = torch.full((b,), s, dtype=torch.int32, device="cuda")
    qt, kn, vn = mk(b, 1, h, d), mk(b, 1, hk, d), mk(b, 1, hk, d)

    def run():
        o, lse = ops.flash_attn_sink_fwd(q, k, v, 0.125, (64, 0), 4)
        grads = ops.flash_attn_sink_bwd(do, q, k, v, o, lse, 0.125, (64, 0), 4)
        w = torch.zeros(b, hk, s, device="cuda")
        ops.flash_attn_paged(q[:, -8:], k, v, None, lens, 0.125, weights_out=w)
        kept, w2, n2 = ops.flash_attn_evict(k, v, w, lens, budget, 4, 32, None, kp, vp, table)
        ot, lt, w2 = ops.flash_attn_paged(qt, kp, vp, table, n2, 0.125, k_new=kn, v_new=vn, weights=w2, weights_out=w2)
        return (o, lse) + tuple(grads) + (kept, n2, ot, lt, w2)

    def fill(seed):
        gg = gen(seed)
        for t in (q, k, v, do, qt, kn, vn):
            t.copy_(randn(gg, *t.shape))

    fill(1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for seed in (2, 3, 4):
        fill(seed)
        want = [t.clone() for t in run()]
        kp0 = kp.clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, x in zip(want, captured):
            assert torch.equal(a, x)
        assert torch.equal(kp, kp0)


def test_a_run_of_them_prompt_evict_decode():
    """Prompt, its last rows' attention as weights, eviction into pages, tokens, eviction in place, tokens: every step
    against the definition on the state that the steps before it left."""
    g = gen(14)
    b, s, h, hk, d, budget = 3, 1500, 8, 2, 128, 400
    dt = torch.bfloat16
    q, k, v = randn(g, b, s, h, d, dtype=dt), randn(g, b, s, hk, d, dtype=dt), randn(g, b, s, hk, d, dtype=dt)
    scale = d ** -0.5
    want = R.attention(q, k, v, scale, (512, 0), 4)
    o, lse = ops.flash_attn_sink_fwd(q, k, v, scale, (512, 0), 4)
    R.close(o, want["o"], want["o_tol"], "prompt")
    lens = torch.tensor([s, s - 7, 300], dtype=torch.int32, device="cuda")
    w = torch.zeros(b, hk, s, device="cuda")
    ops.flash_attn_paged(q[:, -32:], k, v, None, lens, scale, weights_out=w)
    kp, vp, table = pages_of(g, b, budget + 16, 32, hk, d, dt)
    kept, w, n = ops.flash_attn_evict(k, v, w, lens, budget, 4, 64, None, kp, vp, table)
    assert n.tolist() == [budget, budget, 300]
    for step in range(6):
        if step == 3:
            before = w.clone()
            kept, w, n = ops.flash_attn_evict(kp, vp, w, n, budget // 2, 4, 50, block_table=table)
            assert torch.equal(kept.cpu(), R.evict(before, torch.tensor([budget + 3, budget + 3, 303]), w.shape[2], budget // 2, 4, 50)[0])
        qt, kn, vn = randn(g, b, 1, h, d, dtype=dt), randn(g, b, 1, hk, d, dtype=dt), randn(g, b, 1, hk, d, dtype=dt)
        want = R.paged(qt, kp, vp, table, n, scale, (100, 0), 4, kn, vn, w, w)
        o, lse, w = ops.flash_attn_paged(qt, kp, vp, table, n, scale, (100, 0), 4, kn, vn, w, w)
        R.close(o, want["o"], want["o_tol"], "token")
        R.close(lse, want["lse"], want["lse_tol"], "token lse")
        R.close(w, want["weights"], want["weights_tol"], "weights")
        assert torch.equal(kp, want["k_pages"]) and torch.equal(vp, want["v_pages"])
        n += 1


def test_scalars_in_tensors_are_read_at_every_call():
    """A 0-d tensor as the scale or a count that changes between calls: each call takes its value then."""
    g = gen(5)
    q, k, v = randn(g, 1, 40, 2, 64), randn(g, 1, 90, 2, 64), randn(g, 1, 90, 2, 64)
    scale, sinks, left = torch.tensor(0.0625), torch.tensor(0), torch.tensor(7)
    lens = torch.tensor([90], dtype=torch.int32, device="cuda")
    w = torch.rand(1, 2, 90, generator=g, device="cuda")
    for s, n, wl in ((0.0625, 0, 7), (0.25, 3, 7), (0.25, 3, 20)):
        scale.fill_(s), sinks.fill_(n), left.fill_(wl)
        o, lse = ops.flash_attn_sink_fwd(q, k, v, scale, (left, 0), sinks)
        want = ops.flash_attn_sink_fwd(q, k, v, s, (wl, 0), n)
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
        grads = ops.flash_attn_sink_bwd(q, q, k, v, o, lse, scale, (left, 0), sinks)
        assert all(map(torch.equal, grads, ops.flash_attn_sink_bwd(q, q, k, v, o, lse, s, (wl, 0), n)))
        got = ops.flash_attn_paged(q[:, :2], k, v, None, lens, scale, (left, 0), sinks)
        assert all(map(torch.equal, got, ops.flash_attn_paged(q[:, :2], k, v, None, lens, s, (wl, 0), n)))
        got = ops.flash_attn_evict(k, v, w, lens, left, sinks, k_out=torch.zeros_like(k), v_out=torch.zeros_like(v))
        want = ops.flash_attn_evict(k, v, w, lens, wl, n, k_out=torch.zeros_like(k), v_out=torch.zeros_like(v))
        assert all(map(torch.equal, got, want))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("s, ahead, h, hk, d", [(300, 0, 2, 2, 64), (900, 0, 4, 2, 64), (900, 0, 2, 1, 128), (700, 40, 3, 3, 72), (600, 0, 2, 2, 192),
                                                (2500, 0, 16, 16, 128)])
def test_rows_of_few_keys_have_no_rounding_of_the_stored_output(s, ahead, h, hk, d, dtype):
    """The first row of a causal call, which sees one key, has dS = dP - D = 0.  With D from the stored O, dS would be
    off by the rounding of that O, half a step of the type; without it three dot products of d terms in fp32 are
    left (dP of either kernel, D), each off by (d + 2) 2^-24 sum |dO V|, one rounding of D, and what P is off
    times that rounding of O, far below another.  dS is then rounded to the type's least step."""
    g = gen(s + d)
    q, k, v, do = (randn(g, 1, s, n, d, dtype=dtype) for n in (h, hk, hk, h))
    q, do = q[:, ahead:], do[:, ahead:]
    if ahead:  # row 0 sees ahead + 1 keys: all but one far below it
        k[:, :ahead], q[:, 0], k[:, ahead] = -8.0, 8.0, 8.0
    scale = 1 / math.sqrt(d)
    o, lse = ops.flash_attn_sink_fwd(q, k, v, scale, (s, 0), 4)
    dq, _, _ = ops.flash_attn_sink_bwd(do, q, k, v, o, lse, scale, (s, 0), 4)
    grow = lambda t: t[0, ahead].double().abs().repeat_interleave(h // hk, 0)
    dp = (do[0, 0].double().abs() * grow(v)).sum(1, keepdim=True)
    tol = scale * grow(k) * (4 * (d + 2) * 2.0 ** -24 * dp + R.half_step(dtype) * R.LEAST[R.half_step(dtype)])
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # the rounding of dq itself
    R.close(dq[0, 0], torch.zeros_like(tol), tol, (s, h, d, dtype))
