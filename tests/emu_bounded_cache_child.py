"""The bounded-cache calls as `custom` ops of one ByRE module, through the host builds of the runtime and of the
kernel libraries (see emu_session_child, which points the package at them): started by
tests/test_bounded_cache_refusals.py in a process of its own."""
import struct

import emu_session_child as C  # first: it sets where the libraries come from

import torch

import bounded_cache_ref as R
from byteir_amd import brt, ops


def op(api, names, types, blob, fmt):
    """One byre.custom line whose extra_args are the fields of `blob`."""
    extra = ", ".join(f"{x!r} : f32" if isinstance(x, float) else f"{x} : i64" for x in struct.unpack(fmt, blob))
    return (f'    "byre.custom"({", ".join("%" + n for n in names)}) {{callee = "custom", lib_path = "libflash_attn.so", api_name = "{api}", '
            f'version = "2.5.3", extra_args = [{extra}]}} : ({", ".join(types[n] for n in names)}) -> ()\n')


def main():
    g = torch.Generator().manual_seed(31)
    b, s, h, hk, d, budget, page, n_pages = 1, 90, 4, 2, 64, 40, 16, 5
    rn = lambda *shape: torch.randn(shape, generator=g).half()
    t = dict(q=rn(b, s, h, d), k=rn(b, s, hk, d), v=rn(b, s, hk, d), do=rn(b, s, h, d), o=torch.zeros(b, s, h, d).half(), lse=torch.zeros(b, h, s),
             dq=torch.zeros(b, s, h, d).half(), dk=torch.zeros(b, s, hk, d).half(), dv=torch.zeros(b, s, hk, d).half(), dsm=torch.zeros(b, h, 128),
             acc=torch.zeros(b, 128, h, d), rng=torch.zeros(2, dtype=torch.int64), pm=torch.zeros(1),
             w=torch.rand(b, hk, s, generator=g), n=torch.tensor([s], dtype=torch.int32), table=torch.tensor([[3, 0, 4]], dtype=torch.int32),
             kp=rn(n_pages, page, hk, d), vp=rn(n_pages, page, hk, d), w2=torch.zeros(b, hk, 48), n2=torch.zeros(1, dtype=torch.int32),
             kept=torch.zeros(b, hk, budget, dtype=torch.int32), qt=rn(b, 1, h, d), kn=rn(b, 1, hk, d), vn=rn(b, 1, hk, d),
             ot=torch.zeros(b, 1, h, d).half(), lt=torch.zeros(b, h, 1))
    names = {torch.float16: "f16", torch.float32: "f32", torch.int32: "i32", torch.int64: "i64"}
    types = {n: f'memref<{"x".join(str(i) for i in x.shape)}x{names[x.dtype]}, "cuda">' for n, x in t.items()}
    sink = ops.pack_flash_sink_args(t["q"], t["k"], t["v"], t["o"], 0.125, (20, 0), 4)
    evict = ops.pack_flash_evict_args(t["k"], t["v"], t["kp"], t["vp"], b, 0, 3, budget, 4, 8)
    token = ops.pack_flash_paged_args(t["qt"], t["kp"], t["vp"], t["kn"], t["vn"], t["ot"], 0.125, (-1, 0), 0, 3, 2)
    f_sink, f_evict, f_token = "<17qf4qf3q", "<24q", "<23qf8q"

    def module(sink):
        body = op("run_flash_attn_sink_fwd", ["q", "k", "v", "rng", "o", "lse", "pm"], types, sink, f_sink)
        body += op("run_flash_attn_sink_bwd", ["do", "q", "k", "v", "o", "lse", "rng", "dq", "dk", "dv", "dsm", "acc"], types, sink, f_sink)
        body += op("run_flash_attn_evict", ["k", "v", "w", "n", "table", "kp", "vp", "table", "w2", "n2", "kept"], types, evict, f_evict)
        body += op("run_flash_attn_paged", ["qt", "kp", "vp", "kn", "vn", "table", "n2", "ot", "lt", "w2", "w2"], types, token, f_token)
        args = ", ".join(f'%{n} : {types[n]} {{byre.argname = "{n}", byre.argtype = {2 if n in ("o", "ot") else 1}: i32}}' for n in t)
        return f"module attributes {{byre.container_module}} {{\n  func.func @test({args}) attributes {{byre.entry_point}} {{\n{body}    return\n  }}\n}}\n"

    session = brt.Session(device="ROCM")
    session.load_from_memory(module(sink))
    order = list(t)
    arrays = [t[n].numpy() for n in order]
    C.run(session, arrays).close()
    want = R.attention(t["q"], t["k"], t["v"], 0.125, (20, 0), 4, t["do"])
    for n in ("o", "lse", "dq", "dk", "dv"):
        R.close(t[n], want[n], want[n + "_tol"], n)
    kept, n2 = R.evict(t["w"], t["n"], s, budget, 4, 8)
    assert torch.equal(t["kept"], kept) and torch.equal(t["n2"], n2)
    # the cache that eviction left, without the token's row, which came after it
    w2 = torch.zeros_like(t["w2"])
    kp, vp = t["kp"].clone(), t["vp"].clone()
    for c in range(hk):
        src = kept[0, c].long()
        rows = R.rows_of(kp, t["table"], 0, budget)[0][:, c]
        assert torch.equal(rows, t["k"][0, src, c])
        w2[0, c, :budget] = t["w"][0, c, src]
    want = R.paged(t["qt"], kp, vp, t["table"], t["n2"], 0.125, (-1, 0), 0, t["kn"], t["vn"], w2, w2)
    R.close(t["ot"], want["o"], want["o_tol"], "token")
    R.close(t["w2"], want["weights"], want["weights_tol"], "weights")
    session.close()
    bad = brt.Session(device="ROCM")  # a call that the library refuses fails the run instead of ending the process
    bad.load_from_memory(module(sink[:-8] + struct.pack("<q", -3)))
    try:
        C.run(bad, arrays)
    except RuntimeError as e:
        assert "n_sink -3 is negative" in str(e), e
    else:
        raise AssertionError("a negative n_sink ran")
    print("ok bounded cache")


if __name__ == "__main__":
    main()
