"""Embedding tables and linear adapters (quiver_b200.embed): calls side by side, wide ranges,
infinities, float32 results of 16-bit inputs, waits that run out. Against 64-bit computations;
bounds are derived as in test_embed_gpu.py (u = 2^-24, half a step of the result's type)."""
import math
import threading

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


@pytest.fixture(scope="module")
def embed(gpu):
    from quiver_b200 import embed as e
    return e


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, t=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)


def assert_within(got, want, bound, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float((off / bound.clamp(min=1e-300)).nan_to_num(1e9).max()):.3g} "
                           f"of the bound")


def test_threads_with_tables_of_different_sizes(embed):
    """Gradients of narrow and wide tables side by side: their sorts need different amounts of
    shared memory. (Calls of the C ABI with their arguments ready, so that they follow each other
    closely.)"""
    import ctypes as C
    from quiver_b200 import _native
    lib = _native.lib()
    n, dim = 9000, 4
    ids = torch.randint(0, 3, (n,), generator=gen(1), device="cuda")
    up = normal(gen(2), n, dim)
    tables = (3, 2047) * 4  # digits of 2 and of 11 bits
    want = [embed.embedding_grad(up, ids, r) for r in tables]
    torch.cuda.synchronize()
    bad = []

    def work(rows, want):
        s = torch.cuda.Stream()
        size = C.c_size_t()
        _native.check(lib.qv_embedding_grad_workspace(n, rows, dim, C.byref(size)))
        with torch.cuda.stream(s):
            out = torch.empty(rows, dim, device="cuda")
            ws = torch.empty(size.value, dtype=torch.uint8, device="cuda")
        args = (0, 0, up.data_ptr(), dim, 1, ids.data_ptr(), n, rows, dim, C.c_float(1.0),
                out.data_ptr(), dim, ws.data_ptr(), size.value, s.cuda_stream)
        for _ in range(3000):
            if lib.qv_embedding_grad_device(*args) != 0:
                bad.append((rows, lib.qv_last_error()))
                break
        s.synchronize()
        if not torch.equal(out, want):
            bad.append(rows)

    threads = [threading.Thread(target=work, args=a) for a in zip(tables, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad
