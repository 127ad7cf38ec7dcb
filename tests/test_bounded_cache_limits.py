"""The bounded-cache calls at the limits of what they take: windows beyond 32 bits, calls without query rows,
scratch that is short, launches beyond what 32 bits count.  Executed on the host (emu_util)."""
import os
import struct
import subprocess
import sys

import pytest
import torch

import bounded_cache_ref as R
import emu_util as E
from byteir_amd import ops

pytestmark = pytest.mark.skipif(not (os.path.exists(E.LIB) or os.path.exists("/opt/rocm/llvm/bin/clang++")),
                                reason="no host clang to build the emulated library with")


def randn(gen, *shape, dtype=torch.float16):
    return torch.randn(shape, generator=gen).to(dtype)


WIDE = 1 << 32


@pytest.mark.parametrize("window, same", [
    ((WIDE, 0), (-1, 0)), ((WIDE + 3, 0), (-1, 0)), ((7, WIDE), (7, -1)), ((7, WIDE + 2), (7, -1)), ((-1, WIDE), (-1, -1)),
    ((WIDE + 3, WIDE + 1), (-1, -1)), (((1 << 63) - 1, 0), (-1, 0)), ((-WIDE + 5, 0), (-1, 0)), ((7, -(1 << 63) + 1), (7, -1)),
])
def test_windows_beyond_32_bits(window, same):
    """A side that reaches past every key is no bound, however wide; a negative one is none either."""
    gen = torch.Generator().manual_seed(2)
    q, k, v, do = (randn(gen, 1, n, 2, 32) for n in (50, 90, 90, 50))
    want, got = E.sink_fwd(q, k, v, 0.2, same, 3), E.sink_fwd(q, k, v, 0.2, window, 3)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    grads = E.sink_bwd(do, q, k, v, *got, 0.2, window, 3)
    assert all(map(torch.equal, grads, E.sink_bwd(do, q, k, v, *want, 0.2, same, 3)))
    # prompt and token see the same keys
    paged = E.paged(q[:, -2:], k, v, None, torch.tensor([90], dtype=torch.int32), 0.2, window, 3)
    exact = R.attention(q, k, v, 0.2, same, 3, do)
    R.close(got[0], exact["o"], exact["o_tol"], "o")
    R.close(paged[0], exact["o"][:, -2:], exact["o_tol"][:, -2:], "paged o")
    for name, g in zip(("dq", "dk", "dv"), grads):
        R.close(g, exact[name], exact[name + "_tol"], name)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("mode", [1, 2])
def test_no_query_rows_keep_the_weights(paged, mode):
    """seqlen_q = 0: no key's weight grows, so that weights_out is weights (or 0) for the rows in the cache, and
    what lies behind them is left as it was."""
    gen = torch.Generator().manual_seed(3)
    b, hk, d, page, n = 3, 2, 32, 8, 5
    cap = page * n
    k = randn(gen, *((20, page) if paged else (b, cap)), hk, d)
    table = torch.randperm(20, generator=gen)[:b * n].to(torch.int32).view(b, n).contiguous() if paged else None
    lens = torch.tensor([23, -1, cap + 9], dtype=torch.int32)
    q = torch.empty(b, 0, 4, d, dtype=torch.float16)
    w = torch.rand(b, hk, cap, generator=gen)
    before = E.guarded((b, hk, cap), torch.float32).fill_(-7)
    out = E.guarded((b, hk, cap), torch.float32).copy_(before)
    o, lse = E.paged(q, k, k, table, lens, 0.2, (-1, 0), 0, weights=w if mode == 2 else None, weights_out=out)
    assert o.shape == (b, 0, 4, d) and lse.shape == (b, 4, 0)
    want = before.clone()
    for i, rows in enumerate((23, 0, cap)):
        want[i, :, :rows] = w[i, :, :rows] if mode == 2 else 0
    assert torch.equal(out, want)
    if mode == 2:  # in place
        E.paged(q, k, k, table, lens, 0.2, (-1, 0), 0, weights=out, weights_out=out)
        assert torch.equal(out, want)
    need = E.workspace_bytes("paged", ops.pack_flash_paged_args(q, k, k, None, None, o, 0.2, (-1, 0), 0, n if paged else 0, mode), q.dtype)
    assert need == 0


# The scores behind the weights are kept for 256 MiB of rows x capacity at a time, one column tile (32 rows) at least.
SCORES = 256 << 20


def long_cache(gen, b, hk, d, cap, page, dtype=torch.float16):
    """A cache that could hold `cap` rows a sequence, of which the first two pages exist."""
    n = cap // page
    k, v = randn(gen, 2 * b, page, hk, d, dtype=dtype), randn(gen, 2 * b, page, hk, d, dtype=dtype)
    table = torch.full((b, n), -1, dtype=torch.int32)
    table[:, :2] = torch.randperm(2 * b, generator=gen).to(torch.int32).view(b, 2)
    return k, v, table


def weighted(gen, b, sq, h, hk, d, cap, n_new, lens, window, n_sink, room, page=1 << 7):
    """A call with weights in `room(bytes asked for)` bytes of scratch (None: the library allocates) against the definition."""
    k, v, table = long_cache(gen, b, hk, d, cap, page)
    q = randn(gen, b, sq, h, d)
    kn, vn = (randn(gen, b, n_new, hk, d), randn(gen, b, n_new, hk, d)) if n_new else (None, None)
    n = torch.tensor(lens, dtype=torch.int32)
    # the rows in use and some behind them; the rest of a long row of weights is never looked at
    w, out = torch.rand(b, hk, cap, generator=gen), torch.full((b, hk, cap), -7.0)
    short = 2 * page
    want = R.paged(q, k, v, table[:, :2].contiguous(), n, 0.2, window, n_sink, kn, vn, w[:, :, :short].contiguous(), out[:, :, :short].contiguous())
    need = E.workspace_bytes("paged", ops.pack_flash_paged_args(q, k, v, kn, vn, q, 0.2, window, n_sink, table.shape[1], 2), q.dtype)
    ws = None if room is None else E.guarded((room(need),), torch.uint8)
    o, lse = E.paged(q, k, v, table, n, 0.2, window, n_sink, kn, vn, w, out, workspace=ws)
    R.close(o, want["o"], want["o_tol"], "o")
    R.close(lse, want["lse"], want["lse_tol"], "lse")
    R.close(out[:, :, :short], want["weights"], want["weights_tol"], "weights")
    assert bool((out[:, :, short:] == -7).all())
    assert torch.equal(k, want["k_pages"]) and torch.equal(v, want["v_pages"])
    return need


@pytest.mark.parametrize("b, sq, h, hk, cap, n_new, lens, window, n_sink", [
    # launches that end inside a key/value head: tiles 0 1 | 2, 0 | 1 2 of 96 columns
    (1, 24, 8, 2, 1 << 20, 24, [70], (-1, 0), 0),
    # a tile a launch, the second of eight columns
    (1, 40, 1, 1, 1 << 22, 0, [100], (-1, 0), 0),
    # several sequences a launch, the new rows written by the attention itself
    (3, 1, 8, 1, 1 << 22, 1, [200, -1, 33], (-1, 0), 0),
])
def test_scores_that_do_not_fit_the_scratch_at_once(b, sq, h, hk, cap, n_new, lens, window, n_sink):
    gen = torch.Generator().manual_seed(sq)
    need = weighted(gen, b, sq, h, hk, 32, cap, n_new, lens, window, n_sink, lambda n: n)  # exactly what was asked for
    rows, tile = b * h * sq, min(32, h // hk * sq)
    assert rows * cap * 4 > SCORES
    at_once = max(tile, SCORES // (cap * 4))  # rows of a launch
    assert need <= at_once * cap * 4 + 64 * at_once * (32 + 2) * 4  # scores, and the partials of 64 splits


def test_without_memory_ever_fewer_tiles_a_launch():
    """A process that may not allocate what a call asks for: the call falls back to fewer tiles a launch, in the caller's
    scratch when that holds one, and fails with an error when there is no room for one."""
    code = """if True:
        import os, resource, sys
        sys.path[:0] = [%r, %r]
        import torch
        torch.set_num_threads(1)
        import test_bounded_cache_limits as T
        import emu_util as E
        gen = torch.Generator().manual_seed(7)
        args = (1, 24, 8, 2, 32, 1 << 18, 24, [70], (-1, 0), 0)
        need = T.weighted(gen, *args, None)             # everything allocated once
        tile = 32 * (1 << 18) * 4                       # scores of one column tile: 32 MiB
        assert need > 5 * tile
        soft, hard = resource.getrlimit(resource.RLIMIT_AS)
        tight = lambda: resource.setrlimit(resource.RLIMIT_AS, (int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize() + room, hard))
        paged = E.paged
        for room, ws in ((3 * tile, None), (tile // 2, tile), (tile // 2, 2 * tile + 512)):
            def limited(*a, **k):
                tight()
                try:
                    return paged(*a, **k)
                finally:
                    resource.setrlimit(resource.RLIMIT_AS, (soft, hard))
            E.paged = limited
            T.weighted(gen, *args, None if ws is None else lambda n: ws)
        room = tile // 2
        try:
            T.weighted(gen, *args, None)
        except E.EmuFault as e:
            assert "rc 2" in str(e), e                  # out of memory
            print("ok without memory")
    """ % (E.ROOT, os.path.join(E.ROOT, "tests"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "ok without memory" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]


def test_evictions_beyond_a_launch_are_refused():
    """A launch counts its threads in 32 bits, an eviction takes 1024 for a head, and in place for a column slice of one:
    more are refused before anything is launched."""
    def blob(b, hk, d, page=2):  # a dense cache, in place
        return struct.pack("<24q", *[d] * 12, b, hk, d, b, page, 0, b, page, 0, 1, 0, 0)
    # never looked at: one tensor stands for them all
    t, n = torch.zeros(16, dtype=torch.float16), torch.zeros(16, dtype=torch.int32)
    w = torch.zeros(16)
    other = torch.zeros(16, dtype=torch.float16)
    for b, hk, d in ((1 << 22, 1, 8), (1 << 12, 1 << 10, 8), (1 << 12, 64, 256), (1 << 20, 2, 8)):
        with pytest.raises(E.EmuFault, match="too large"):
            E._call("evict", [t, t, w, n, None, t, t, None, w, n, n], blob(b, hk, d), torch.float16)
    with pytest.raises(E.EmuFault, match="too large"):  # into another cache
        E._call("evict", [t, t, w, n, None, other, other, None, w.clone(), n, n], blob(1 << 22, 1, 8), torch.float16)


def test_a_broadcast_workspace_is_refused(monkeypatch):
    """Its elements say nothing of the bytes behind it."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)  # where CPU tensors say they lie
    plan = (lambda *a: pytest.fail("launched"), b"", 1, 1 << 20)
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 21, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="workspace must be dense"):
            ops._launch(plan, b"", torch.zeros(1), ws)
