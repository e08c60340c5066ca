"""Layer norm, dropout and the linear cross entropy refuse bad arguments before
any device work (no GPU needed)."""
import ctypes

import pytest


class FakeBuf:
    handle = 16  # never dereferenced on these paths

    def __init__(self, n_bytes):
        self.n_bytes = n_bytes


@pytest.fixture(scope="module")
def lib():
    from nx_vulkan_b200 import _native, build
    build.build()
    return _native.load()


P = ctypes.c_void_p(16)  # never dereferenced on these paths


def test_null_arguments(lib):
    for k in range(6):
        a = [P] * 6
        a[k] = None
        assert lib.nxv_layer_norm(*a, 2, 4, 1e-5, 0, b"layer_norm.spv") == -1
    for k in (0, 1, 2, 4, 5, 6, 7, 8):  # 3 is the optional workspace
        a = [P] * 9
        a[k] = None
        assert lib.nxv_layer_norm_grad(*a, 2, 4, 0, b"layer_norm_grad.spv") == -1
    assert lib.nxv_dropout(None, P, 4, 0.1, 1, 0, 0, b"dropout.spv") == -1
    assert lib.nxv_dropout(P, P, 4, 0.1, 1, 0, 0, None) == -1
    for k in (0, 1, 3, 4, 5):
        a = [P] * 6
        a[k] = None
        assert lib.nxv_linear_cross_entropy(*a, 2, 3, 4, 0, 8, b"linear_cross_entropy.spv") == -1
    for k in (0, 1, 3, 4, 5, 6, 7):
        a = [P] * 8
        a[k] = None
        assert lib.nxv_linear_cross_entropy_grad(*a, 2, 3, 4, 0, 8,
                                                 b"linear_cross_entropy_grad.spv") == -1


def test_unknown_kernel_names(lib):
    bad = b"reduce.spv"
    assert lib.nxv_layer_norm(*[P] * 6, 2, 4, 1e-5, 0, bad) == -2
    assert lib.nxv_layer_norm_grad(*[P] * 9, 2, 4, 0, bad) == -2
    assert lib.nxv_dropout(P, P, 4, 0.1, 1, 0, 0, bad) == -2
    assert lib.nxv_linear_cross_entropy(*[P] * 6, 2, 3, 4, 0, 8, bad) == -2
    assert lib.nxv_linear_cross_entropy_grad(*[P] * 8, 2, 3, 4, 0, 8, bad) == -2


def test_values_out_of_range(lib):
    nan, inf = float("nan"), float("inf")
    ln = lambda rows, cols, eps, dt: lib.nxv_layer_norm(*[P] * 6, rows, cols, eps, dt,  # noqa: E731
                                                        b"layer_norm.spv")
    for args in ((2, 0, 1e-5, 0), (2, (1 << 28) + 1, 1e-5, 0), (2, 4, -1e-5, 0), (2, 4, nan, 0), (2, 4, inf, 0), (2, 4, 1e-5, 3)):
        assert ln(*args) == -3
    assert lib.nxv_layer_norm_grad(*[P] * 9, 2, 0, 0, b"layer_norm_grad.spv") == -3
    assert lib.nxv_layer_norm_grad(*[P] * 9, 2, (1 << 28) + 1, 0, b"layer_norm_grad.spv") == -3
    assert lib.nxv_layer_norm_grad(*[P] * 9, 2, 4, 3, b"layer_norm_grad.spv") == -3
    for n, p, off, dt in ((4, -0.1, 0, 0), (4, 1.1, 0, 0), (4, nan, 0, 0), (4, 0.1, 0, 3),
                          ((1 << 32) + 1, 0.1, 0, 0), (4, 0.1, (1 << 32) - 3, 0),
                          (4, 0.1, (1 << 64) - 2, 0)):
        assert lib.nxv_dropout(P, P, n, p, 1, off, dt, b"dropout.spv") == -3
    for n, v, d, dt, ib in ((2, 0, 4, 0, 8), (2, 3, 0, 0, 8), (2, 3, 4, 1, 8), (2, 3, 4, 3, 8),
                            (2, 3, 4, 0, 2), (1 << 31, 3, 4, 0, 8), (2, 1 << 31, 4, 0, 8),
                            (2, 3, 1 << 31, 0, 8)):
        assert lib.nxv_linear_cross_entropy(*[P] * 6, n, v, d, dt, ib,
                                            b"linear_cross_entropy.spv") == -3
        assert lib.nxv_linear_cross_entropy_grad(*[P] * 8, n, v, d, dt, ib,
                                                 b"linear_cross_entropy_grad.spv") == -3
    assert lib.nxv_linear_cross_entropy_workspace(2, 0, 4, 0, 0) == 0
    assert lib.nxv_linear_cross_entropy_workspace(2, 3, 4, 0, 0) > 0
    assert lib.nxv_layer_norm_grad_workspace(5, 7, 0) >= 2 * 7 * 4
    assert lib.nxv_layer_norm_grad_workspace(5, 7, 3) == 0


def test_the_mirror_refuses_too(lib):
    from nx_vulkan_b200 import vulkan as nxv
    b = FakeBuf
    assert nxv.layer_norm(b(32), b(16), b(16), 2, 4, -1.0) == ("error", "bad_op")
    assert nxv.layer_norm(b(32), b(16), b(16), 2, 4, float("nan")) == ("error", "bad_op")
    assert nxv.layer_norm(b(32), b(16), b(16), 2, 4, dtype="f16") == ("error", "bad_op")
    assert nxv.layer_norm(b(31), b(16), b(16), 2, 4) == ("error", "size_mismatch")
    assert nxv.layer_norm(b(32), b(16), b(12), 2, 4) == ("error", "size_mismatch")
    assert nxv.layer_norm(b(32), b(16), b(16), 2, 4, out=(b(32), b(8), b(4))) == ("error", "size_mismatch")
    assert nxv.layer_norm(b(0), b(0), b(0), 2, 0) == ("error", "bad_op")
    assert nxv.layer_norm_grad(b(32), b(32), b(16), b(4), b(8), 2, 4) == ("error", "size_mismatch")
    assert nxv.layer_norm_grad(b(32), b(32), b(16), b(8), b(8), 2, 4, dtype="x") == ("error", "bad_op")
    assert nxv.dropout(b(16), 1.5, 1) == ("error", "bad_op")
    assert nxv.dropout(b(16), 0.5, -1) == ("error", "bad_op")
    assert nxv.dropout(b(16), 0.5, 1, offset=(1 << 32) - 3) == ("error", "bad_op")
    assert nxv.dropout(b(15), 0.5, 1) == ("error", "size_mismatch")
    assert nxv.dropout(b(16), 0.5, 1, out=b(12)) == ("error", "size_mismatch")
    ce = nxv.linear_cross_entropy
    assert ce(b(32), b(48), b(16), 2, 3, 4, dtype="f64") == ("error", "bad_op")
    assert ce(b(32), b(48), b(16), 2, 3, 4, index_bytes=2) == ("error", "bad_op")
    assert ce(b(32), b(48), b(16), 2, 0, 4) == ("error", "bad_op")
    assert ce(b(32), b(44), b(16), 2, 3, 4) == ("error", "size_mismatch")
    assert ce(b(32), b(48), b(8), 2, 3, 4) == ("error", "size_mismatch")
    cg = nxv.linear_cross_entropy_grad
    assert cg(b(4), b(32), b(48), b(16), b(8), 2, 3, 4) == ("error", "size_mismatch")
    assert cg(b(8), b(32), b(48), b(16), b(8), 2, 3, 4, out=(b(32), b(40))) == ("error", "size_mismatch")


def test_limits_of_the_workspaces_and_of_dim(lib):
    from nx_vulkan_b200 import vulkan as nxv
    big = (1 << 24) + 1
    assert lib.nxv_linear_cross_entropy(*[P] * 6, 2, 3, big, 0, 8, b"linear_cross_entropy.spv") == -3
    assert lib.nxv_linear_cross_entropy_grad(*[P] * 8, 2, 3, big, 2, 8, b"linear_cross_entropy_grad.spv") == -3
    b = FakeBuf
    assert nxv.linear_cross_entropy(b(8 * big), b(12 * big), b(16), 2, 3, big) == ("error", "bad_op")
    for args in ((2, 0, 4), (2, 3, big), ((1 << 32) + 2, 3, 4), (2, 3, 4, "f64"), (2, 3, 4, "f16")):
        assert nxv.linear_cross_entropy_workspace(*args) == 0
    for args in ((2, 0), ((1 << 32) + 2, 4), (2, (1 << 28) + 1), (2, 4, "f16")):
        assert nxv.layer_norm_grad_workspace(*args) == 0
