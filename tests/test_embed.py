"""Argument checks of the embedding and adapter entry points that need no GPU: the Python layer's,
and the C ABI's workspace and size checks, which are pure host code."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from quiver_b200 import _native, embed  # noqa: E402


def grad_workspace(n, rows, dim):
    size = C.c_size_t()
    _native.check(_native.lib().qv_embedding_grad_workspace(n, rows, dim, C.byref(size)))
    return size.value


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(3, 4), torch.zeros(5, 4)
    ids = torch.zeros(3, dtype=torch.long)
    for f in (lambda: embed.linear(x, w), lambda: embed.linear("x", w),
              lambda: embed.linear(x, None), lambda: embed.linear_preact(x, w),
              lambda: embed.linear_grad(torch.zeros(3, 5), x, w),
              lambda: embed.embedding_lookup(w, ids), lambda: embed.embedding_lookup([1.0], ids),
              lambda: embed.embedding_grad(x, ids, 7), lambda: embed.Adapter(w),
              lambda: embed.Adapter(None)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            f()


def test_no_gradient_path_for_cpu_tensors():
    w = torch.zeros(5, 4, requires_grad=True)
    with pytest.raises(ValueError, match="CUDA tensor"):
        embed.linear(torch.zeros(3, 4), w)
    with pytest.raises(ValueError, match="CUDA tensor"):
        embed.embedding_lookup(w, torch.zeros(3, dtype=torch.long))


def test_activation_names():
    assert set(embed.ACTIVATIONS) == {"none", "relu", "gelu", "gelu_tanh", "silu"}
    for name in ("GELU", "tanh", "", None):
        with pytest.raises(ValueError, match="unknown activation"):
            embed._activation_code(name)


def test_grad_workspace_sizes():
    assert grad_workspace(0, 100, 8) == 0
    assert grad_workspace(100, 0, 8) == 0
    last = 0
    for n in (1, 1000, 8192, 8193, 100_000, 2_000_000):
        size = grad_workspace(n, 50_000, 64)
        assert size >= 8 * n and size >= last
        last = size
    with pytest.raises(ValueError, match="dimension"):
        grad_workspace(10, 10, 0)
    with pytest.raises(ValueError, match="dimension"):
        grad_workspace(10, 10, 65537)
    with pytest.raises(ValueError, match="2\\^31"):
        grad_workspace(10, 2 ** 31, 8)
    with pytest.raises(ValueError, match="2\\^31"):
        grad_workspace(2 ** 31, 10, 8)


def test_null_arguments():
    lib = _native.lib()
    size = C.c_size_t()
    for call in (lambda: lib.qv_linear_workspace(0, None, C.byref(size)),
                 lambda: lib.qv_linear_grad_workspace(0, None, C.byref(size)),
                 lambda: lib.qv_embedding_grad_workspace(1, 1, 1, None),
                 lambda: lib.qv_linear_device(0, None, None, 0, None),
                 lambda: lib.qv_linear_grad_device(0, None, None, 0, None),
                 lambda: lib.qv_flat_lookup_device(None, 1, None, 0, 1.0, None, 8, None)):
        with pytest.raises(ValueError, match="null"):
            _native.check(call())


def test_struct_layouts_match_the_header():
    """The ctypes mirrors have the C structs' sizes (three or two 32-bit fields, then 64-bit ones)."""
    assert C.sizeof(_native.qv_linear) == 16 + 14 * 8
    assert C.sizeof(_native.qv_linear_grad) == 8 + 16 * 8


def test_result_memory_checks():
    t = torch.zeros(6, 8)
    with pytest.raises(ValueError, match="share memory with x"):
        embed._apart(t[2:4], x=t)
    with pytest.raises(ValueError, match="share memory with b"):
        embed._apart(t, a=torch.zeros(3), b=t[5, 7:])
    embed._apart(t[:3], x=t[3:], y=None, z=t[:0])
    with pytest.raises(ValueError, match="contiguous"):
        embed._check_out(t.t(), (8, 6), torch.float32, t.device)
    with pytest.raises(ValueError, match="expected"):
        embed._check_out(t, (8, 6), torch.float32, t.device)
    with pytest.raises(ValueError, match="gradient"):
        embed._check_out(t.clone().requires_grad_(), (6, 8), torch.float32, t.device)


def test_rows_copies_only_what_it_must():
    t = torch.zeros(6, 8)
    assert embed._rows(t) is t
    assert embed._rows(t[:, 2:5]).data_ptr() == t[:, 2:5].data_ptr()
    assert embed._rows(t[:1].expand(6, 8)).stride() == (8, 1)
    assert embed._rows(t.t()).is_contiguous()
    assert embed._rows(t[::2]).data_ptr() == t.data_ptr()
