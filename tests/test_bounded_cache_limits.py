"""The bounded-cache calls at the limits of what they take: windows beyond 32 bits, calls without query rows,
scratch that is short, launches beyond what 32 bits count.  Executed on the host (emu_util)."""
import os

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
