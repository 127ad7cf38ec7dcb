"""The bounded-cache calls at the limits of what they take, on the GPU (the same on the host: test_bounded_cache_limits)."""
import pytest
import torch

import bounded_cache_ref as R
from byteir_amd import ops

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float16):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def test_windows_beyond_32_bits():
    g = gen(1)
    q, k, v, do = (randn(g, 1, n, 2, 64) for n in (80, 300, 300, 80))
    for window, same in (((1 << 32, 0), (-1, 0)), (((1 << 32) + 3, 1 << 32), (-1, -1)), ((9, (1 << 32) + 1), (9, -1))):
        want, got = (ops.flash_attn_sink_fwd(q, k, v, 0.125, w, 3) for w in (same, window))
        assert all(map(torch.equal, got, want))
        grads, other = (ops.flash_attn_sink_bwd(do, q, k, v, *got, 0.125, w, 3) for w in (same, window))
        assert all(map(torch.equal, grads, other))


@pytest.mark.parametrize("paged", [False, True])
def test_no_query_rows_keep_the_weights(paged):
    g = gen(2)
    b, hk, cap = 3, 2, 2100
    k = randn(g, *((400, 21) if paged else (b, cap)), hk, 64)
    table = torch.randperm(400, generator=g, device="cuda")[:300].to(torch.int32).view(b, 100).contiguous() if paged else None
    lens = torch.tensor([1500, -1, cap], dtype=torch.int32, device="cuda")
    w, out = torch.rand(b, hk, cap, generator=g, device="cuda"), torch.full((b, hk, cap), -7.0, device="cuda")
    ops.flash_attn_paged(randn(g, b, 0, 4, 64), k, k, table, lens, 0.125, weights=w, weights_out=out)
    want = torch.full_like(out, -7.0)
    want[0, :, :1500], want[2] = w[0, :, :1500], w[2]
    assert torch.equal(out, want)
    ops.flash_attn_paged(randn(g, b, 0, 4, 64), k, k, table, lens, 0.125, weights_out=out)
    want[0, :, :1500], want[2] = 0, 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("b, sq, h, hk, n_new, lens", [
    (12, 1, 16, 4, 1, [300, 1, -1, 77, 1000, 0, 1023, 512, 31, 32, 33, 900]),  # 768 MiB of scores, several sequences a launch
    (2, 24, 8, 2, 0, [700, 20]),                                               # tiles of a head in two launches
])
def test_scores_that_do_not_fit_the_scratch_at_once(b, sq, h, hk, n_new, lens):
    g = gen(b)
    cap, page, d, short = 1 << 20, 512, 64, 1024
    k, v = randn(g, 2 * b, page, hk, d), randn(g, 2 * b, page, hk, d)
    table = torch.full((b, cap // page), -1, dtype=torch.int32, device="cuda")
    table[:, :2] = torch.randperm(2 * b, generator=g, device="cuda").to(torch.int32).view(b, 2)
    q = randn(g, b, sq, h, d)
    kn, vn = (randn(g, b, n_new, hk, d), randn(g, b, n_new, hk, d)) if n_new else (None, None)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    w, out = torch.rand(b, hk, cap, generator=g, device="cuda"), torch.full((b, hk, cap), -7.0, device="cuda")
    need = ops.flash_attn_workspace_bytes("paged", q.dtype, ops.pack_flash_paged_args(q, k, v, kn, vn, q, 0.125, (-1, 0), 0, cap // page, 2))
    assert b * h * sq * cap * 4 > 384 << 20 and need < 272 << 20
    want = R.paged(q, k, v, table[:, :2].contiguous(), n, 0.125, (-1, 0), 0, kn, vn, w[:, :, :short].contiguous(), out[:, :, :short].contiguous())
    o, lse, _ = ops.flash_attn_paged(q, k, v, table, n, 0.125, k_new=kn, v_new=vn, weights=w, weights_out=out)
    R.close(o, want["o"], want["o_tol"], "o")
    R.close(lse, want["lse"], want["lse_tol"], "lse")
    R.close(out[:, :, :short], want["weights"], want["weights_tol"], "weights")
    assert bool((out[:, :, short:] == -7).all())
    assert torch.equal(k, want["k_pages"]) and torch.equal(v, want["v_pages"])


def test_a_call_of_several_launches_is_captured_and_replayed():
    """Replayed three times on new inputs, with eager calls between, in scratch of its own."""
    g = gen(3)
    b, h, hk, d, cap, page = 12, 16, 4, 64, 1 << 20, 512
    k, v = torch.empty(2 * b, page, hk, d, device="cuda", dtype=torch.float16), torch.empty(2 * b, page, hk, d, device="cuda", dtype=torch.float16)
    table = torch.full((b, cap // page), -1, dtype=torch.int32, device="cuda")
    table[:, :2] = torch.arange(2 * b, device="cuda", dtype=torch.int32).view(b, 2)
    q, kn, vn = (torch.empty(b, 1, n, d, device="cuda", dtype=torch.float16) for n in (h, hk, hk))
    n = torch.randint(0, 1000, (b,), generator=g, device="cuda").to(torch.int32)
    w, out = torch.zeros(b, hk, cap, device="cuda"), torch.zeros(b, hk, cap, device="cuda")

    def run():
        return ops.flash_attn_paged(q, k, v, table, n, 0.125, k_new=kn, v_new=vn, weights=w, weights_out=out)

    def fill():
        for t in (q, k, v, kn, vn):
            t.copy_(randn(g, *t.shape))
        w[:, :, :1024] = torch.rand(b, hk, 1024, generator=g, device="cuda")

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for _ in range(3):
        fill()
        want = [t.clone() for t in run()]
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(map(torch.equal, captured, want))
