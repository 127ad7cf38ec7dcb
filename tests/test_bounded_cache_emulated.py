"""Attention with a window and sinks, over a paged cache, and eviction, executed on the host lane by lane against
their definitions in 64 bits; tensors end at (or begin behind) a protected page, so that an access outside
them is a reported fault.  The tolerances are those of bounded_cache_ref."""
import os

import numpy as np
import pytest
import torch

import bounded_cache_ref as R
import emu_util as E

pytestmark = pytest.mark.skipif(not (os.path.exists(E.LIB) or os.path.exists("/opt/rocm/llvm/bin/clang++")),
                                reason="no host clang to build the emulated library with")


def guard(t, at_end=True):
    return E.guarded(tuple(t.shape), t.dtype, at_end).copy_(t)


def randn(gen, *shape, dtype=torch.float16, at_end=True):
    return guard(torch.randn(shape, generator=gen).to(dtype), at_end)


SINK_CASES = [
    # b, sq, sk, h, h_k, d, window, n_sink
    (1, 130, 130, 2, 1, 64, (40, 0), 4),       # the usual four, grouped heads
    (1, 300, 300, 2, 2, 128, (30, 0), 1),      # tuned kernels at 128: sinks in tile 0, windows far from it
    (2, 90, 333, 2, 2, 32, (50, 3), 70),       # a chunk against a longer cache, sinks over two tiles
    (1, 290, 290, 4, 2, 96, (17, 0), 33),      # a head_dim without a tuned kernel
    (1, 70, 20, 1, 1, 64, (9, 0), 4),          # more rows than keys: the first rows see nothing
    (1, 1, 200, 4, 4, 128, (20, 0), 4),        # one row
    (1, 150, 150, 1, 1, 64, (0, 0), 2),        # a window of the row's own key
    (1, 100, 260, 2, 2, 40, (-1, 0), 4),       # no left side: sinks change nothing
    (1, 64, 200, 1, 1, 64, (25, -1), 300),     # no right side, sinks beyond the keys
    (1, 520, 520, 1, 1, 64, (600, 0), 4),      # rows of more than 512 keys: D of the first rows in a launch of its own
    (1, 516, 530, 1, 1, 40, (550, 2), 0),      # the same, columns behind head_dim
    (1, 140, 140, 2, 1, 256, (33, 0), 5),      # the widest head
    (1, 200, 0, 1, 1, 64, (9, 0), 4),          # no keys
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", SINK_CASES)
def test_sink_forward_and_backward(case, dtype):
    b, sq, sk, h, hk, d, window, ns = case
    gen = torch.Generator().manual_seed(sq * 7 + sk + d)
    at_end = d != 96
    q, do = (randn(gen, b, sq, h, d, dtype=dtype, at_end=at_end) for _ in range(2))
    k, v = (randn(gen, b, sk, hk, d, dtype=dtype, at_end=at_end) for _ in range(2))
    scale = 1 / np.sqrt(d)
    G = lambda s, t=dtype: E.guarded(s, t, at_end)
    o, lse = E.sink_fwd(q, k, v, scale, window, ns, out=(G(q.shape), G((b, h, sq), torch.float32)))
    dq, dk, dv = E.sink_bwd(do, q, k, v, o, lse, scale, window, ns,
                            out=(G(q.shape), G(k.shape), G(v.shape), G((b, h, -(-sq // 128) * 128), torch.float32)))
    want = R.attention(q, k, v, scale, window, ns, do)
    for name, got in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        R.close(got, want[name], want[name + "_tol"], (name, case))


def test_sink_keys_that_no_row_sees_may_hold_anything():
    gen = torch.Generator().manual_seed(5)
    q, do = (randn(gen, 1, 40, 2, 64) for _ in range(2))
    k, v = (randn(gen, 1, 400, 2, 64) for _ in range(2))
    k[:, 3:340] = float("nan")   # sinks are 0..2, the first row's window begins at 360 - 20
    v[:, 3:340] = float("inf")
    o, lse = E.sink_fwd(q, k, v, 0.125, (20, 0), 3)
    dq, dk, dv = E.sink_bwd(do, q, k, v, o, lse, 0.125, (20, 0), 3)
    want = R.attention(q, k, v, 0.125, (20, 0), 3, do)
    for name, got in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        R.close(got, want[name], want[name + "_tol"], name)


def test_sink_strided_storage_and_workspace():
    """[b, h, s, d] storage, scratch of the caller's for the key split, the group's partials and the sinks' shares."""
    gen = torch.Generator().manual_seed(6)
    q, do = (randn(gen, 1, 4, 260, 64).transpose(1, 2) for _ in range(2))
    k, v = (randn(gen, 1, 2, 1500, 64).transpose(1, 2) for _ in range(2))
    from byteir_amd import ops
    args = (0.125, (1200, 0), 40)
    blob = ops.pack_flash_sink_args(q, k, v, q, *args)
    o_ws = E.workspace_bytes("sink_fwd", blob, q.dtype)
    b_ws = E.workspace_bytes("sink_bwd", blob, q.dtype)
    assert o_ws > 0 and b_ws > 0
    o, lse = torch.empty_like(q), torch.empty(1, 4, 260)
    E.sink_fwd(q, k, v, *args, out=(o, lse), workspace=guard(torch.full((o_ws,), 255, dtype=torch.uint8)))
    o2, lse2 = E.sink_fwd(q, k, v, *args, out=(torch.empty_like(q), torch.empty(1, 4, 260)))
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    got = E.sink_bwd(do, q, k, v, o, lse, *args, workspace=guard(torch.full((b_ws,), 255, dtype=torch.uint8)))
    again = E.sink_bwd(do, q, k, v, o, lse, *args)
    want = R.attention(q, k, v, *args, do)
    R.close(o, want["o"], want["o_tol"], "o")
    R.close(lse, want["lse"], want["lse_tol"], "lse")
    for name, x, y in zip(("dq", "dk", "dv"), got, again):
        assert torch.equal(x, y)
        R.close(x, want[name], want[name + "_tol"], name)


def pages_of(gen, b, cap, page, hk, d, dtype, spare=2):
    """A pool whose pages a shuffled table names -> k, v, table."""
    n = -(-cap // page)
    k, v = (randn(gen, b * n + spare, page, hk, d, dtype=dtype) for _ in range(2))
    table = guard(torch.randperm(b * n + spare, generator=gen)[:b * n].to(torch.int32).view(b, n))
    return k, v, table


PAGED_CASES = [
    # lens, capacity, page, sq, n_new, h, h_k, d, window, n_sink, weights
    ([300, 0, 77], 320, 16, 1, 1, 8, 2, 128, (-1, 0), 0, False),
    ([1500, 31], 2048, 64, 1, 1, 4, 2, 64, (-1, 0), 0, True),     # split over workgroups
    ([900, 2000, 5], 2048, 7, 1, 0, 2, 2, 64, (100, 0), 4, True),  # a page size that fits nothing, window and sinks
    ([700, -1, 40], 800, 100, 3, 3, 6, 2, 40, (33, 0), 40, True),   # an idle sequence, drafted rows
    ([0, 1, 2], 64, 1, 4, 0, 4, 4, 32, (-1, 0), 0, True),          # fewer keys than rows
    ([200, 333], 384, 24, 20, 20, 4, 1, 96, (-1, 0), 0, True),     # several column tiles: the new rows by their own kernel
    ([250, 100], 256, 32, 70, 70, 1, 1, 256, (50, 2), 3, False),   # rows behind the capacity, tiles of one head
    ([400], 512, 256, 2, 9, 2, 1, 64, (3, 0), 1, True),            # a window that does not reach the first new row
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", PAGED_CASES)
def test_paged(case, dtype):
    lens, cap, page, sq, n_new, h, hk, d, window, ns, weighted = case
    b = len(lens)
    gen = torch.Generator().manual_seed(cap + page + d)
    k, v, table = pages_of(gen, b, cap, page, hk, d, dtype)
    q = randn(gen, b, sq, h, d, dtype=dtype)
    kn, vn = (randn(gen, b, n_new, hk, d, dtype=dtype) for _ in range(2)) if n_new else (None, None)
    full = table.shape[1] * page
    w = guard(torch.rand((b, hk, full), generator=gen)) if weighted else None
    w_out = guard(torch.full((b, hk, full), -7.0)) if weighted else None
    n = guard(torch.tensor(lens, dtype=torch.int32))
    scale = 1 / np.sqrt(d)
    want = R.paged(q, k, v, table, n, scale, window, ns, kn, vn, w, w_out)
    o, lse = E.paged(q, k, v, table, n, scale, window, ns, kn, vn, w, w_out, out=(E.guarded(q.shape, dtype), E.guarded((b, h, sq), torch.float32)))
    R.close(o, want["o"], want["o_tol"], ("o", case))
    R.close(lse, want["lse"], want["lse_tol"], ("lse", case))
    assert torch.equal(k, want["k_pages"]) and torch.equal(v, want["v_pages"])
    if weighted:
        R.close(w_out, want["weights"], want["weights_tol"], ("weights", case))


def test_paged_dense_cache_is_the_same_as_pages():
    gen = torch.Generator().manual_seed(9)
    k, v = (randn(gen, 2, 100, 2, 64) for _ in range(2))
    q, n = randn(gen, 2, 1, 4, 64), torch.tensor([100, 63], dtype=torch.int32)
    a = E.paged(q, k, v, None, n, 0.125, (40, 0), 2)
    pool = torch.stack([t.reshape(2, 5, 20, 2, 64) for t in (k, v)])
    table = torch.tensor([[4, 0, 6, 1, 9], [3, 2, 8, 7, 5]], dtype=torch.int32)
    kp, vp = torch.zeros(2, 10, 20, 2, 64, dtype=k.dtype)
    kp[table.long()], vp[table.long()] = pool[0], pool[1]
    c = E.paged(q, kp, vp, table, n, 0.125, (40, 0), 2)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


def test_paged_absent_pages_and_what_nobody_sees():
    """Page numbers outside the pool hide their keys; rows behind the last key, outside the window or on no
    table hold NaN; new rows that fall on an absent page are dropped."""
    gen = torch.Generator().manual_seed(10)
    k, v, table = pages_of(gen, 2, 160, 16, 2, 64, torch.float16)
    n = torch.tensor([150, 145], dtype=torch.int32)
    table[0, 3], table[0, 7], table[1, 9], table[1, 0] = -1, k.shape[0], 1 << 30, -(1 << 31)
    q = randn(gen, 2, 2, 4, 64)
    kn, vn = (randn(gen, 2, 2, 2, 64) for _ in range(2))
    used = torch.zeros(k.shape[:2], dtype=torch.bool)
    for i in range(2):
        for j in list(range(3)) + list(range(int(n[i]) + 2 - 2 - 60, int(n[i]))):
            if 0 <= int(table[i, j // 16]) < k.shape[0]:
                used[table[i, j // 16], j % 16] = True
    k[~used], v[~used] = float("nan"), float("nan")
    w_out = torch.zeros(2, 2, 160)
    want = R.paged(q, k, v, table, n, 0.125, (60, 0), 3, kn, vn, None, w_out)
    o, lse = E.paged(q, k, v, table, n, 0.125, (60, 0), 3, kn, vn, None, w_out)
    R.close(o, want["o"], want["o_tol"], "o")
    R.close(lse, want["lse"], want["lse_tol"], "lse")
    R.close(w_out, want["weights"], want["weights_tol"], "weights")
    assert torch.equal(k.view(torch.int16), want["k_pages"].view(torch.int16)) and torch.equal(v.view(torch.int16), want["v_pages"].view(torch.int16))


EVICT_CASES = [
    # lens, source rows, budget, n_sink, n_recent, h_k, d, page (0: dense), page of the output
    ([300, 50, 51, -1], 300, 50, 4, 10, 2, 64, 16, 32),
    ([100, 97], 100, 96, 0, 0, 1, 128, 0, 7),
    ([2500], 2500, 1200, 1, 100, 1, 40, 64, 0),
    ([64, 65], 70, 64, 30, 34, 2, 32, 8, 8),   # nothing competes
    ([9, 1, 0], 9, 1, 0, 0, 1, 8, 3, 1),
    ([500], 400, 100, 2, 3, 1, 256, 50, 50),   # a length beyond the capacity counts as the capacity
]


def evict_setup(case, gen, dtype):
    lens, rows, budget, ns, nr, hk, d, page, page_out = case
    b = len(lens)
    if page:
        k, v, table = pages_of(gen, b, rows, page, hk, d, dtype)
        cap = table.shape[1] * page
    else:
        k, v, table, cap = randn(gen, b, rows, hk, d, dtype=dtype), randn(gen, b, rows, hk, d, dtype=dtype), None, rows
    w = torch.rand((b, hk, cap), generator=gen)
    w = torch.where(torch.rand((b, hk, cap), generator=gen) < 0.4, (w * 4).floor() / 4, w)  # equal weights, zeros
    special = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0, -1.5, 1e-42])
    at = torch.rand((b, hk, cap), generator=gen) < 0.1
    w[at] = special[torch.randint(0, 6, (int(at.sum()),), generator=gen)]
    return b, k, v, table, cap, guard(w), guard(torch.tensor(lens, dtype=torch.int32))


def moved(pages, table, kept, i, c):
    src = kept[i, c][kept[i, c] >= 0].long()
    x, ok = R.rows_of(pages, table, i, int(src.max()) + 1 if len(src) else 0)
    return x[src, c]


@pytest.mark.parametrize("case", EVICT_CASES)
def test_evict_into_another_cache(case):
    gen = torch.Generator().manual_seed(case[1])
    lens, rows, budget, ns, nr, hk, d, page, page_out = case
    b, k, v, table, cap, w, n = evict_setup(case, gen, torch.bfloat16)
    if page_out:
        ko, vo, to = pages_of(gen, b, budget, page_out, hk, d, torch.bfloat16)
        cap_out = to.shape[1] * page_out
    else:
        ko, vo, to, cap_out = randn(gen, b, budget + 3, hk, d, dtype=torch.bfloat16), randn(gen, b, budget + 3, hk, d, dtype=torch.bfloat16), None, budget + 3
    w_out, n_out, kept = guard(torch.full((b, hk, cap_out), -3.0)), guard(torch.zeros(b, dtype=torch.int32)), guard(torch.zeros(b, hk, budget, dtype=torch.int32))
    ko0, vo0, k0, w0 = ko.clone(), vo.clone(), k.clone(), w.clone()
    E.evict(k, v, w, n, budget, ns, nr, table, ko, vo, to, w_out, n_out, kept)
    want, n_want = R.evict(w, n, cap, budget, ns, nr)
    assert torch.equal(kept, want) and torch.equal(n_out, n_want)
    assert torch.equal(k, k0) and torch.equal(w.view(torch.int32), w0.view(torch.int32)) and n.tolist() == lens
    for i in range(b):
        for c in range(hk):
            src = want[i, c][want[i, c] >= 0].long()
            ko0_rows = R.rows_of(ko, to, i, len(src))[0][:, c]
            assert torch.equal(ko0_rows, moved(k, table, want, i, c)) and torch.equal(R.rows_of(vo, to, i, len(src))[0][:, c], moved(v, table, want, i, c))
            assert torch.equal(w_out[i, c, :len(src)].view(torch.int32), w[i, c, src].view(torch.int32)) and bool((w_out[i, c, len(src):] == -3).all())
            # rows behind the kept ones are as they were
            rest = slice(len(src), cap_out)
            assert torch.equal(R.rows_of(ko, to, i, cap_out)[0][rest, c], R.rows_of(ko0, to, i, cap_out)[0][rest, c])


@pytest.mark.parametrize("case", EVICT_CASES)
def test_evict_in_place(case):
    gen = torch.Generator().manual_seed(case[1] + 1)
    lens, rows, budget, ns, nr, hk, d, page, _ = case
    b, k, v, table, cap, w, n = evict_setup(case, gen, torch.float16)
    kept = guard(torch.zeros(b, hk, budget, dtype=torch.int32))
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    want, n_want = R.evict(w, n, cap, budget, ns, nr)
    E.evict(k, v, w, n, budget, ns, nr, table, k, v, table, w, n, kept)
    assert torch.equal(kept, want) and torch.equal(n, n_want)
    for i in range(b):
        for c in range(hk):
            src = want[i, c][want[i, c] >= 0].long()
            for new, old in ((k, k0), (v, v0)):
                after, before = R.rows_of(new, table, i, cap)[0][:, c], R.rows_of(old, table, i, cap)[0][:, c]
                assert torch.equal(after[:len(src)], before[src]) and torch.equal(after[len(src):], before[len(src):])
            assert torch.equal(w[i, c, :len(src)].view(torch.int32), w0[i, c, src].view(torch.int32))
            assert torch.equal(w[i, c, len(src):].view(torch.int32), w0[i, c, len(src):].view(torch.int32))


def test_a_run_of_them_prompt_evict_decode():
    """A prompt under window and sinks, its last rows' attention as weights, eviction into pages, then tokens one by
    one over what is left -- each step against the definition, on the state that the steps before it left."""
    gen = torch.Generator().manual_seed(21)
    b, s, h, hk, d, budget = 2, 150, 4, 2, 64, 60
    q, k, v = randn(gen, b, s, h, d), randn(gen, b, s, hk, d), randn(gen, b, s, hk, d)
    want = R.attention(q, k, v, 0.125, (64, 0), 4)
    o, lse = E.sink_fwd(q, k, v, 0.125, (64, 0), 4)
    R.close(o, want["o"], want["o_tol"], "prompt")
    lens = torch.full((b,), s, dtype=torch.int32)
    w = torch.zeros(b, hk, s)
    E.paged(q[:, -16:].contiguous(), k, v, None, lens, 0.125, (-1, 0), 0, weights_out=w)
    kp, vp, table = pages_of(gen, b, budget + 8, 16, hk, d, torch.float16)
    w2, n2, kept = torch.zeros(b, hk, table.shape[1] * 16), torch.zeros(b, dtype=torch.int32), torch.zeros(b, hk, budget, dtype=torch.int32)
    E.evict(k, v, w, lens, budget, 4, 16, None, kp, vp, table, w2, n2, kept)
    assert torch.equal(kept, R.evict(w, lens, s, budget, 4, 16)[0]) and n2.tolist() == [budget] * b
    for _ in range(3):
        qt, kn, vn = randn(gen, b, 1, h, d), randn(gen, b, 1, hk, d), randn(gen, b, 1, hk, d)
        want = R.paged(qt, kp, vp, table, n2, 0.125, (-1, 0), 0, kn, vn, w2, w2)
        o, lse = E.paged(qt, kp, vp, table, n2, 0.125, (-1, 0), 0, kn, vn, w2, w2)  # weights on top of themselves
        R.close(o, want["o"], want["o_tol"], "token")
        R.close(w2, want["weights"], want["weights_tol"], "weights")
        assert torch.equal(kp, want["k_pages"])
        n2 += 1
