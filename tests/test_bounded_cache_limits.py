"""The bounded-cache calls at the limits of what they take: windows beyond 32 bits, calls without query rows,
scratch that is short, launches beyond what 32 bits count.  Executed on the host (emu_util)."""
import os

import pytest
import torch

import bounded_cache_ref as R
import emu_util as E

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
