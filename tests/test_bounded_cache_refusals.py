"""What the bounded-cache calls refuse, without a GPU: at the C entry points (the host build of the library: an
error code and a reason, nothing launched) and in byteir_amd.ops (ValueError before the library is called);
and the calls as `custom` ops of a ByRE module, run through the host build of the runtime."""
import os
import struct
import subprocess
import sys

import pytest
import torch

import emu_util as E
from byteir_amd import ops

pytestmark = pytest.mark.skipif(not (os.path.exists(E.LIB) or os.path.exists("/opt/rocm/llvm/bin/clang++")),
                                reason="no host clang to build the emulated library with")

H = torch.float16


def sink_tensors(b=1, sq=8, sk=8, h=2, hk=1, d=32, dtype=H):
    q, do = torch.zeros(b, sq, h, d, dtype=dtype), torch.zeros(b, sq, h, d, dtype=dtype)
    return q, torch.zeros(b, sk, hk, d, dtype=dtype), torch.zeros(b, sk, hk, d, dtype=dtype), do


@pytest.mark.parametrize("change,why", [
    (dict(n_sink=-1), "n_sink -1 is negative"), (dict(scale=0.0), "softmax_scale 0 is not positive"), (dict(scale=-0.5), "not positive"),
    (dict(scale=float("nan")), "not positive"), (dict(scale=float("inf")), "not positive"), (dict(d=36), "head_dim 36"), (dict(d=264), "head_dim 264"),
    (dict(h=3, hk=2), "must be a multiple of h_k"),
])
def test_sink_refusals(change, why):
    args = dict(n_sink=4, scale=0.5)
    args.update({k: v for k, v in change.items() if k in args})
    q, k, v, do = sink_tensors(**{k: v for k, v in change.items() if k not in args})
    with pytest.raises(E.EmuFault, match=why):
        E.sink_fwd(q, k, v, args["scale"], (4, 0), args["n_sink"])
    lse = torch.zeros(q.shape[0], q.shape[2], q.shape[1])
    with pytest.raises(E.EmuFault, match=why):
        E.sink_bwd(do, q, k, v, torch.zeros_like(q), lse, args["scale"], (4, 0), args["n_sink"])


def test_sink_refuses_lengths_that_32_bits_do_not_add():
    q, k, v, _ = sink_tensors()
    blob = ops.pack_flash_sink_args(q, k, v, q, 0.5, (4, 0), 4)
    at = 17 * 8 + 4  # seqlen_q, seqlen_k
    for sq, sk in ((1 << 29, 8), (8, 1 << 29), (1 << 28, (1 << 28) + 1)):
        with pytest.raises(E.EmuFault, match="too large"):
            E._call("sink_fwd", [None] * 7, blob[:at] + struct.pack("<2q", sq, sk) + blob[at + 16:], H)


def test_windows_wider_than_everything_are_none():
    """Window sides at the limits of their field."""
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, n, 2, 32, generator=gen).half() for n in (40, 70, 70))
    want = E.sink_fwd(q, k, v, 0.2, (-1, -1), 3)
    for window in ((70, 40), ((1 << 31) - 1, (1 << 31) - 1), (69, 39)):
        got = E.sink_fwd(q, k, v, 0.2, window, 3)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_sink_refuses_dropout_bad_types_and_null_tensors():
    q, k, v, _ = sink_tensors()
    o, lse = torch.zeros_like(q), torch.zeros(1, 2, 8)
    blob = ops.pack_flash_args(q, k, v, o, 0.5, (4, 0), 0.1) + struct.pack("<q", 4)
    with pytest.raises(E.EmuFault, match="dropout is not supported with sinks"):
        E._call("sink_fwd", [q, k, v, None, o, lse, None], blob, H)
    blob = ops.pack_flash_sink_args(q, k, v, o, 0.5, (4, 0), 4)
    with pytest.raises(E.EmuFault, match="null tensor"):
        E._call("sink_fwd", [q, None, v, None, o, lse, None], blob, H)
    assert E.lib().flash_attn_sink_fwd_checked(None, None, 1, None) == -1
    assert E.lib().flash_attn_sink_fwd_workspace_bytes(blob, 3) == 0  # not a storage type


def paged_blob(**change):
    x = dict(b=2, h=4, hk=2, d=64, new=1, scale=0.125, sq=1, pages=8, page=16, max_pages=4, wl=-1, wr=0, sink=0, mode=0, stride=64)
    x.update(change)
    return struct.pack("<23q", *[x["stride"]] * 18, x["b"], x["h"], x["hk"], x["d"], x["new"]) + struct.pack("<f", x["scale"]) + \
        struct.pack("<8q", x["sq"], x["pages"], x["page"], x["max_pages"], x["wl"], x["wr"], x["sink"], x["mode"])


@pytest.mark.parametrize("change,why", [
    (dict(b=-1), "negative"), (dict(hk=0), "zero dimension"), (dict(hk=3), "multiple of h_k"), (dict(d=60), "head_dim 60"), (dict(d=512), "head_dim 512"),
    (dict(stride=4), "not a multiple of 8"), (dict(page=0), "bad page counts"), (dict(pages=-1), "bad page counts"), (dict(max_pages=-1), "bad page counts"),
    (dict(max_pages=1 << 28), r"more than 2\^30 rows"), (dict(max_pages=0, pages=1), "2 sequences in a cache of 1"), (dict(sq=-1), "bad seqlen_q"),
    (dict(new=-1), "seqlen_knew"), (dict(sink=-1), "n_sink"), (dict(mode=3), "weights mode"), (dict(scale=0.0), "not positive"),
    (dict(scale=float("inf")), "not positive"), (dict(sq=0), "new rows without query rows"), (dict(sq=1 << 29), "too large"),
    (dict(b=1 << 22, h=1024, hk=1024), "too large"), (dict(pages=(1 << 31)), "bad page counts"), (dict(page=1 << 28), "too large"),
    (dict(new=1 << 30), "too large"),
])
def test_paged_refusals(change, why):
    # the reason comes before any tensor is looked at
    with pytest.raises(E.EmuFault, match=why):
        E._call("paged", [None] * 11, paged_blob(**change), H)


def test_paged_null_and_misaligned_tensors():
    t = torch.zeros(4096, dtype=H)
    n, table, lse, w = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(8), torch.zeros(2, 2, 64)
    full = [t, t, t, t, t, table, n, t, lse, w, w]
    for i in (0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10):
        with pytest.raises(E.EmuFault, match="null tensor"):
            E._call("paged", full[:i] + [None] + full[i + 1:], paged_blob(mode=2), H)
    for i in (0, 1, 2, 3, 4, 7):
        with pytest.raises(E.EmuFault, match="16-byte aligned"):
            E._call("paged", full[:i] + [t[1:]] + full[i + 1:], paged_blob(mode=2), H)


def evict_blob(**change):
    x = dict(b=2, hk=2, d=64, np=8, page=16, mp=4, npo=8, pageo=16, mpo=4, budget=20, sink=4, recent=4, stride=64, stride_out=64)
    x.update(change)
    return struct.pack("<24q", *[x["stride"], x["stride"], x["stride_out"], x["stride_out"]] * 3, *(x[n] for n in
                       ("b", "hk", "d", "np", "page", "mp", "npo", "pageo", "mpo", "budget", "sink", "recent")))


@pytest.mark.parametrize("change,why", [
    (dict(b=-1), "negative"), (dict(d=4), "head_dim 4"), (dict(stride=12), "multiple of 8"), (dict(page=0), "cache: bad page counts"),
    (dict(pageo=0), "output cache: bad page counts"), (dict(mp=0, np=1), "sequences in a cache"), (dict(budget=0), "budget 0"),
    (dict(budget=65), "does not fit the output cache"), (dict(sink=-1), "n_sink"), (dict(sink=10, recent=11), "do not fit the budget"),
    (dict(sink=21, recent=0), "do not fit the budget"), (dict(recent=-1), "n_recent"),
    (dict(b=1 << 20, hk=16, budget=60), "too large"),
])
def test_evict_refusals(change, why):
    with pytest.raises(E.EmuFault, match=why):
        E._call("evict", [None] * 11, evict_blob(**change), H)


def test_evict_half_in_place():
    k, v, ko, vo = (torch.zeros(8, 16, 2, 64, dtype=H) for _ in range(4))
    w, w2, n, table = torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    kept, other = torch.zeros(2, 2, 20, dtype=torch.int32), table.clone()
    full = [k, v, w, n, table, ko, vo, table, w2, n.clone(), kept]
    for swap, blob, why in (({5: k}, {}, "cache's own"), ({6: v}, {}, "cache's own"), ({5: k, 6: v, 7: other}, {}, "cache's own"),
                            ({5: k, 6: v}, dict(stride_out=128), "cache's own"), ({5: k, 6: v}, dict(mpo=3), "cache's own"),
                            ({8: w}, {}, "in place only together"), ({2: None}, {}, "null tensor"), ({10: None}, {}, "null tensor")):
        with pytest.raises(E.EmuFault, match=why):
            E._call("evict", [swap.get(i, t) for i, t in enumerate(full)], evict_blob(**blob), H)


def raises(fn, *args, match="", **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_python_calls_check_their_tensors():
    q, k, v, do = sink_tensors()
    o, lse = torch.zeros_like(q), torch.zeros(1, 2, 8)
    f, g = ops.flash_attn_sink_fwd, ops.flash_attn_sink_bwd
    raises(f, q, k, v, 0.5, match="device tensor required")
    raises(f, q.float(), k, v, 0.5, match="float32 is not supported")
    raises(f, q, k.bfloat16(), v, 0.5, match="one storage type")
    raises(f, q[0], k, v, 0.5, match="4-d")
    raises(f, q.transpose(2, 3), k, v, 0.5, match="dense head_dim")
    raises(f, q, k, v[:, :4], 0.5, match="do not fit together")
    raises(f, q, k, v, 0.5, out=(o[:, :4], lse), match="o must be")
    raises(f, q, k, v, 0.5, out=(o, lse.transpose(1, 2).contiguous().transpose(1, 2)), match="lse must be dense")
    raises(g, do[:, :4], q, k, v, o, lse, 0.5, match="dout must be")
    raises(g, do, q, k, v, o, lse.double(), 0.5, match="lse must be")
    raises(g, do, q, k, v, o, lse, 0.5, match="device tensor required")
    kp, n, table = torch.zeros(8, 16, 2, 32, dtype=H), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32)
    p = ops.flash_attn_paged
    raises(p, q, kp, kp, table, n, 0.5, match="device tensor required")
    raises(p, q, kp, kp, table.long(), n, 0.5, match="block_table must be")
    raises(p, q, kp, kp, table[:, ::2], n, 0.5, match="block_table must be dense")
    raises(p, q, kp, kp, None, n, 0.5, match="1 sequences, but a dense cache of 8")
    raises(p, q, kp, kp, table, n.long(), 0.5, match="seqlens_k must be")
    raises(p, q, kp, kp[:4], table, n, 0.5, match="do not fit together")
    raises(p, q, kp, kp, table, n, 0.5, k_new=kp[:1, :1], match="given together")
    raises(p, q, kp[:1].expand(8, 16, 2, 32), kp, table, n, 0.5, k_new=kp[:1, :1], v_new=kp[:1, :1], match="broadcast view")
    raises(p, q, kp, kp, table, n, 0.5, weights=torch.zeros(1, 2, 64), match="without weights_out")
    raises(p, q, kp, kp, table, n, 0.5, weights_out=torch.zeros(1, 2, 63), match="weights_out must be")
    w, e = torch.zeros(1, 2, 64), ops.flash_attn_evict
    raises(e, kp, kp, w, n, 10, block_table=table, match="device tensor required")
    raises(e, kp, kp, w, n, 0, block_table=table, match="budget 0 is not positive")
    raises(e, kp, kp, w, n, -3, block_table=table, match="budget -3 is not positive")
    raises(e, kp, kp, w, n, 10, match="1 sequences, but a dense cache of 8")
    raises(e, kp, kp, w, n, 10, block_table=table, k_out=kp, match="given together")
    raises(e, kp, kp, w, n, 10, block_table=table, out_table=table, match="out_table without k_out")
    raises(e, kp, kp, w[:, :, :60], n, 10, block_table=table, match="weights must be")
    raises(e, kp, kp, w, n, 10, block_table=table, kept=torch.zeros(1, 2, 9, dtype=torch.int32), match="kept must be")
    raises(e, kp, kp, w, n, 10, block_table=table, k_out=kp[..., :16], v_out=kp[..., :16], match="do not fit k")


def test_custom_ops_of_a_module_run_on_the_host():
    """A prompt and its gradient, eviction of its cache into pages and a token over them, as one ByRE module."""
    E.lib()
    child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "emu_bounded_cache_child.py")
    r = subprocess.run([sys.executable, child], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "ok bounded cache" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
