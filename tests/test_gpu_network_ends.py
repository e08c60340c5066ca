"""Layer norm, dropout and the linear cross entropy, with their gradients,
against their formulas in 64 bits.

Tolerances.  u is half a step of the arithmetic's type (f32 2^-24, f64 2^-53)
and h half a step of the result's type (bf16 2^-8).  A sum of k numbers added
by t threads in turn and then in a tree is off by at most (k / t + 12) u times
the sum of their magnitudes.  The tensor cores add 16 products into an f32
accumulator at a time and may truncate, one step (2^-23 of the running sum's
magnitude) per addition: (K / 16 + 8) 2^-23 times the sum of the products'
magnitudes, six times as many additions for f32's six partial products."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"f32": 2.0 ** -24, "f64": 2.0 ** -53, "bf16": 2.0 ** -24}
H = {"f32": 2.0 ** -24, "f64": 2.0 ** -53, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(autouse=True)
def _stream(nxv, torch):
    """The library's work on torch's stream, so that both see each other's results."""
    from nx_vulkan_b200 import _native
    _native.load().nxv_set_stream(torch.cuda.current_stream().cuda_stream or 1)
    yield
    torch.cuda.synchronize()
    _native.load().nxv_set_stream(None)


def dt(torch, name):
    return {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16}[name]


def stat(torch, name):
    return torch.float64 if name == "f64" else torch.float32


def wrap(nxv, t):
    assert t.is_contiguous()
    return nxv.wrap_tensor(t)


def ok(r):
    from nx_vulkan_b200 import _native
    assert r[0] == "ok", (r, _native.last_error())
    return r[1]


def within(torch, got, want, tol):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol) & ~(torch.isnan(got) & torch.isnan(want)) & ~(got == want)
    if bad.any():
        i = int(bad.reshape(-1).nonzero()[0])
        t = torch.as_tensor(tol, device=got.device).expand(got.shape).reshape(-1)[i]
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off, first at {i}: "
                             f"{float(got.reshape(-1)[i])} want {float(want.reshape(-1)[i])} tol {float(t)}")


def place(torch, t, shift):
    """A copy of t that starts `shift` elements after a 256-byte boundary, and its surroundings."""
    room = torch.full((t.numel() + shift + 64,), 7.0, device="cuda", dtype=t.dtype)
    v = room[shift:shift + t.numel()].view(t.shape)
    v.copy_(t)
    return v, room


# ---- layer norm ---------------------------------------------------------------

NORM_SHAPES = [(1, 1), (1, 2), (4, 7), (5, 32), (9, 33), (3, 256), (7, 1000), (2, 1023), (300, 129),
               (3, 4096), (2, 5001), (7, 5003), (2, 8192), (3, 12289), (1, 16384), (2, 20000), (1, 40001), (3, 70001),
               (600, 64), (1200, 33), (700, 1025), (500, 20003),
               (2500, 3), (2400, 257), (2400, 1000), (5000, 104), (2400, 5001),
               (3, 14329), (3, 14343), (2, 28667), (2, 28681), (2, 30001), (2, 57337), (2, 57361)]


def norm_run(nxv, torch, x, g, b, eps, name, y=None):
    r, c = x.shape
    y = torch.full_like(x, 3.0) if y is None else y
    m = torch.full((r,), 5.0, device="cuda", dtype=stat(torch, name))
    s = torch.full_like(m, 5.0)
    out = tuple(wrap(nxv, t) for t in (y, m, s))
    ok(nxv.layer_norm(wrap(nxv, x), wrap(nxv, g), wrap(nxv, b), r, c, eps, dtype=name, out=out))
    return y, m, s


def norm_check(torch, name, x, g, b, eps, y, m, s):
    X, G, B = x.double(), g.double(), b.double()
    c = x.shape[1]
    k = 128 * U[name]  # at most 40 elements a thread, 12 levels, and the formula's own roundings
    M = X.mean(1, keepdim=True)
    S = 1 / ((X - M).square().mean(1, keepdim=True) + eps).sqrt()
    size = X.abs().mean(1, keepdim=True)
    within(torch, m[:, None], M, k * size + U[name] * M.abs())
    # the centred values are off by the mean's error, and rstd by what that and the sum add
    within(torch, s[:, None], S, S * k * (1 + size * S))
    xh = (X - M) * S
    within(torch, y, xh * G + B,
           H[name] * (xh * G + B).abs() + k * (G.abs() * (xh.abs() + size * S) * (1 + size * S) + B.abs()))


@pytest.mark.parametrize("name", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_layer_norm(nxv, torch, name, shape):
    torch.manual_seed(shape[0] * 31 + shape[1])
    d = dt(torch, name)
    x = (torch.randn(shape, device="cuda") * 2 + 0.5).to(d)
    g, b = torch.randn(shape[1], device="cuda").to(d), torch.randn(shape[1], device="cuda").to(d)
    norm_check(torch, name, x, g, b, 1e-5, *norm_run(nxv, torch, x, g, b, 1e-5, name))


@pytest.mark.parametrize("name", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("cols", [64, 1000, 1001])
@pytest.mark.parametrize("shift", [0, 1, 3, 8])
def test_layer_norm_at_any_address(nxv, torch, name, cols, shift):
    torch.manual_seed(cols + shift)
    d = dt(torch, name)
    x, _ = place(torch, torch.randn(5, cols, device="cuda").to(d), shift)
    g, _ = place(torch, torch.randn(cols, device="cuda").to(d), shift + 1)
    b, _ = place(torch, torch.randn(cols, device="cuda").to(d), shift)
    y, room = place(torch, torch.zeros(5, cols, device="cuda", dtype=d), shift)
    out = norm_run(nxv, torch, x, g, b, 1e-5, name, y=y)
    norm_check(torch, name, x, g, b, 1e-5, *out)
    assert bool((room[:shift] == 7).all()) and bool((room[shift + 5 * cols:] == 7).all())


def test_layer_norm_special_rows(nxv, torch):
    """A constant row, a row with a large mean, a NaN, an infinity: each stays its row's own."""
    x = torch.randn(6, 300, device="cuda")
    x[1] = 4.0
    x[2] += 4096.0
    x[3, 7] = float("nan")
    x[4, 299] = float("inf")
    g, b = torch.ones(300, device="cuda"), torch.zeros(300, device="cuda")
    y, m, s = norm_run(nxv, torch, x, g, b, 1e-5, "f32")
    keep = [0, 1, 2, 5]
    norm_check(torch, "f32", x[keep], g, b, 1e-5, y[keep], m[keep], s[keep])
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[4]).all())
    assert bool((y[1] == 0).all())  # 300 * 4 and its mean are exact


@pytest.mark.parametrize("cols", [48, 999, 40001])
def test_layer_norm_in_place(nxv, torch, cols):
    x = torch.randn(3, cols, device="cuda")
    g, b = torch.randn(cols, device="cuda"), torch.randn(cols, device="cuda")
    want = norm_run(nxv, torch, x, g, b, 1e-5, "f32")[0].clone()
    assert torch.equal(norm_run(nxv, torch, x, g, b, 1e-5, "f32", y=x)[0], want)


def grad_run(nxv, torch, dy, x, g, m, s, name, dx=None, workspace=None):
    r, c = x.shape
    dx = torch.full_like(x, 3.0) if dx is None else dx
    dg, db = torch.full_like(g, 3.0), torch.full_like(g, 3.0)
    out = tuple(wrap(nxv, t) for t in (dx, dg, db))
    ok(nxv.layer_norm_grad(*(wrap(nxv, t) for t in (dy, x, g, m, s)), r, c, dtype=name, out=out,
                           workspace=workspace))
    return dx, dg, db


def grad_inputs(torch, name, r, c, seed=0):
    torch.manual_seed(seed + r * 31 + c)
    d = dt(torch, name)
    x = (torch.randn(r, c, device="cuda") * 2 + 0.5).to(d)
    dy, g = torch.randn(r, c, device="cuda").to(d), torch.randn(c, device="cuda").to(d)
    X = x.double()
    m = X.mean(1)
    s = 1 / ((X - m[:, None]).square().mean(1) + 1e-5).sqrt()
    return dy, x, g, m.to(stat(torch, name)), s.to(stat(torch, name))


def grad_check(torch, name, dy, x, g, m, s, dx, dg, db):
    DY, X, G, M, S = (t.double() for t in (dy, x, g, m[:, None], s[:, None]))
    r, c = x.shape
    k = 128 * U[name]
    xh, w = (X - M) * S, DY * G
    a, q = w.mean(1, keepdim=True), (w * xh).mean(1, keepdim=True)
    want = S * (w - a - xh * q)
    size = S * (w.abs() + w.abs().mean(1, keepdim=True) + xh.abs() * (w * xh).abs().mean(1, keepdim=True))
    within(torch, dx, want, H[name] * want.abs() + k * size)
    # at most r / 128 + 1 rows a thread, then 2400 / 32 partial rows a thread and 5 levels, 4 roundings a term
    kk = (r / 128 + 1 + 2400 / 32 + 9) * U[name]
    within(torch, dg, (DY * xh).sum(0), H[name] * (DY * xh).sum(0).abs() + kk * (DY * xh).abs().sum(0))
    within(torch, db, DY.sum(0), H[name] * DY.sum(0).abs() + kk * DY.abs().sum(0))


@pytest.mark.parametrize("name", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_layer_norm_grad(nxv, torch, name, shape):
    a = grad_inputs(torch, name, *shape)
    out = grad_run(nxv, torch, *a, name)
    grad_check(torch, name, *a, *out)
    again = grad_run(nxv, torch, *a, name)
    assert all(torch.equal(p, q) for p, q in zip(out, again))


@pytest.mark.parametrize("name", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("shift", [1, 4])
def test_layer_norm_grad_at_any_address(nxv, torch, name, shift):
    a = [place(torch, t, shift)[0] for t in grad_inputs(torch, name, 9, 1000)]
    dx, room = place(torch, torch.zeros_like(a[1]), shift + 1)
    grad_check(torch, name, *a, *grad_run(nxv, torch, *a, name, dx=dx))
    assert bool((room[:shift + 1] == 7).all()) and bool((room[shift + 1 + 9000:] == 7).all())


@pytest.mark.parametrize("name", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("cols", [1, 2, 3, 5, 9])
def test_layer_norm_of_short_rows_at_any_address(nxv, torch, name, cols):
    """Rows shorter than 16 bytes in a tensor that starts between boundaries."""
    for shift in (1, 3):
        dy, x, g, m, s = (place(torch, t, shift)[0] for t in grad_inputs(torch, name, 70, cols))
        dx, room = place(torch, torch.zeros_like(x), shift)
        grad_check(torch, name, dy, x, g, m, s, *grad_run(nxv, torch, dy, x, g, m, s, name, dx=dx))
        assert bool((room[:shift] == 7).all()) and bool((room[shift + 70 * cols:] == 7).all())
        y, room = place(torch, torch.zeros_like(x), shift)
        norm_check(torch, name, x, g, g, 1e-5, *norm_run(nxv, torch, x, g, g, 1e-5, name, y=y))
        assert bool((room[:shift] == 7).all()) and bool((room[shift + 70 * cols:] == 7).all())


@pytest.mark.parametrize("name", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("shape", [(5, 100), (700, 1000), (4, 40001)], ids=str)
def test_layer_norm_grad_of_small_values(nxv, torch, name, shape):
    """Rows of size 1e-18 and eps = 0: rstd's cube would overflow f32, no gradient does."""
    dy, x, g, _, _ = grad_inputs(torch, name, *shape)
    x = x * 1e-18
    X = x.double()
    m = X.mean(1)
    s = 1 / (X - m[:, None]).square().mean(1).sqrt()
    m, s = m.to(stat(torch, name)), s.to(stat(torch, name))
    grad_check(torch, name, dy, x, g, m, s, *grad_run(nxv, torch, dy, x, g, m, s, name))


@pytest.mark.parametrize("cols", [48, 999, 40001])
@pytest.mark.parametrize("which", [0, 1])
def test_layer_norm_grad_in_place(nxv, torch, cols, which):
    a = list(grad_inputs(torch, "f32", 5, cols))
    want = [t.clone() for t in grad_run(nxv, torch, *a, "f32")]
    got = grad_run(nxv, torch, *a, "f32", dx=a[which])
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_layer_norm_no_rows(nxv, torch):
    e = torch.empty(0, 5, device="cuda")
    v, z = torch.ones(5, device="cuda"), torch.empty(0, device="cuda")
    norm_run(nxv, torch, e, v, v, 1e-5, "f32")
    _, dg, db = grad_run(nxv, torch, e, e, v, z, z, "f32")
    assert bool((dg == 0).all()) and bool((db == 0).all())


def test_layer_norm_past_32_bits(nxv, torch):
    """More than 2^31 elements: the last rows are right, and the weights' sums see them."""
    r, c = (1 << 17) + 5, 16392
    x = torch.empty(r, c, device="cuda", dtype=torch.bfloat16).normal_()
    g, b = torch.randn(c, device="cuda").bfloat16(), torch.randn(c, device="cuda").bfloat16()
    y, m, s = norm_run(nxv, torch, x, g, b, 1e-5, "bf16")
    for part in (slice(0, 3), slice(r - 3, r)):
        norm_check(torch, "bf16", x[part], g, b, 1e-5, y[part], m[part], s[part])
    dy = torch.zeros_like(x)
    dy[:2], dy[-2:] = torch.randn(2, c, device="cuda"), torch.randn(2, c, device="cuda")
    dx, dg, db = grad_run(nxv, torch, dy, x, g, m, s, "bf16", dx=y)
    ends = [0, 1, r - 2, r - 1]
    grad_check(torch, "bf16", dy[ends], x[ends], g, m[ends], s[ends], dx[ends], dg, db)


def test_layer_norm_grad_against_differences(nxv, torch):
    """Central differences of sum(dy * y) along a random direction of (x, gamma, beta), in f64:
    truncation h^2 / 6 times third derivatives of order 1, rounding 2^-53 / h."""
    r, c, h = 4, 50, 2.0 ** -12
    torch.manual_seed(1)
    x, dy = (torch.randn(r, c, device="cuda", dtype=torch.float64) for _ in range(2))
    g, b = (torch.randn(c, device="cuda", dtype=torch.float64) for _ in range(2))
    _, m, s = norm_run(nxv, torch, x, g, b, 1e-5, "f64")
    dx, dg, db = grad_run(nxv, torch, dy, x, g, m, s, "f64")
    ex, eg, eb = torch.randn_like(x), torch.randn_like(g), torch.randn_like(b)
    f = lambda t: (dy * norm_run(nxv, torch, x + t * ex, g + t * eg, b + t * eb, 1e-5, "f64")[0]).sum()  # noqa: E731
    want = (f(h) - f(-h)) / (2 * h)
    got = (dx * ex).sum() + (dg * eg).sum() + (db * eb).sum()
    assert abs(float(got - want)) <= 1e-4 * float((dx * ex).abs().sum())


# ---- dropout --------------------------------------------------------------------

def mask_of(nxv, seed, first, n, p):
    """Which stream elements first .. first + n - 1 the library's uniform generator leaves >= p."""
    u = np.frombuffer(ok(nxv.download_binary(ok(nxv.uniform(first + n, seed)), 4 * (first + n))), np.float32)
    return u[first:].astype(np.float64) >= p


@pytest.mark.parametrize("name", ["f32", "f64", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 3, 8, 17, 1000, 4097, 100003])
@pytest.mark.parametrize("offset", [0, 1, 6, 1001])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(nxv, torch, name, n, offset, p):
    seed = n * 7 + offset
    x = torch.randn(n, device="cuda", dtype=torch.float64).to(dt(torch, name))
    y = torch.full_like(x, 9.0)
    ok(nxv.dropout(wrap(nxv, x), p, seed, offset=offset, dtype=name, out=wrap(nxv, y)))
    keep = torch.from_numpy(mask_of(nxv, seed, offset, n, p)).cuda()
    scale = 1 / (1 - p) if p < 1 else 0.0
    w = stat(torch, name)
    want = torch.where(keep, (x.to(w) * torch.tensor(scale, dtype=w)).to(x.dtype), torch.zeros_like(x))
    assert torch.equal(y, want)  # one product and one rounding: bit for bit


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [1, 2, 5])
def test_dropout_at_any_address_and_in_place(nxv, torch, name, shift):
    x, _ = place(torch, torch.randn(1000, device="cuda").to(dt(torch, name)), shift)
    aligned = x.clone()
    y = torch.empty_like(aligned)
    ok(nxv.dropout(wrap(nxv, aligned), 0.3, 5, offset=11, dtype=name, out=wrap(nxv, y)))
    z, room = place(torch, torch.zeros_like(aligned), shift)
    ok(nxv.dropout(wrap(nxv, x), 0.3, 5, offset=11, dtype=name, out=wrap(nxv, z)))
    assert torch.equal(y, z)
    assert bool((room[:shift] == 7).all()) and bool((room[shift + 1000:] == 7).all())
    h = wrap(nxv, x)
    ok(nxv.dropout(h, 0.3, 5, offset=11, dtype=name, out=h))
    assert torch.equal(x, y)


def test_dropout_in_parts_is_dropout_of_the_whole(nxv, torch):
    x = torch.randn(5000, device="cuda")
    y, z = torch.empty_like(x), torch.empty_like(x)
    ok(nxv.dropout(wrap(nxv, x), 0.2, 77, offset=3, out=wrap(nxv, y)))
    for a, b in ((0, 1), (1, 1234), (1234, 5000)):
        ok(nxv.dropout(wrap(nxv, x[a:b]), 0.2, 77, offset=3 + a, out=wrap(nxv, z[a:b])))
    assert torch.equal(y, z)


def test_dropout_drops_nan_and_infinities(nxv, torch):
    x = torch.full((4096,), float("nan"), device="cuda")
    x[1::2] = float("-inf")
    y = torch.empty_like(x)
    ok(nxv.dropout(wrap(nxv, x), 0.5, 3, out=wrap(nxv, y)))
    keep = torch.from_numpy(mask_of(nxv, 3, 0, 4096, 0.5)).cuda()
    assert bool((y[~keep] == 0).all()) and not bool(torch.isfinite(y[keep]).any())


def test_dropout_at_the_end_of_the_stream(nxv, torch):
    """The stream's last elements: counters up to 2^31 - 1 and no wrap."""
    def words(ctr, key):
        a, b = ctr, 0
        for _ in range(10):
            prod = a * 0xD256D193
            a, b = (prod >> 32) ^ key ^ b, prod & 0xFFFFFFFF
            key = (key + 0x9E3779B9) & 0xFFFFFFFF
        return a, b
    n = 37
    first = (1 << 32) - n
    x = torch.ones(n, device="cuda")
    y = torch.empty_like(x)
    ok(nxv.dropout(wrap(nxv, x), 0.5, 42, offset=first, out=wrap(nxv, y)))
    want = [2.0 if (words(i >> 1, 42)[i & 1] >> 8) >= 1 << 23 else 0.0 for i in range(first, first + n)]
    assert y.tolist() == want
    assert nxv.dropout(wrap(nxv, x), 0.5, 42, offset=first + 1) == ("error", "bad_op")


def test_dropout_past_32_bits(nxv, torch):
    """More than 2^32 bytes and 2^31 elements: the end of the whole is the end in parts."""
    n = (1 << 31) + 1037
    x = torch.full((n,), 1.5, device="cuda", dtype=torch.bfloat16)
    y, z = torch.empty_like(x), torch.empty(2000, device="cuda", dtype=torch.bfloat16)
    ok(nxv.dropout(wrap(nxv, x), 0.25, 9, offset=5, dtype="bf16", out=wrap(nxv, y)))
    ok(nxv.dropout(wrap(nxv, x[:2000]), 0.25, 9, offset=5 + n - 2000, dtype="bf16", out=wrap(nxv, z)))
    assert torch.equal(y[-2000:], z) and 1300 < int((z != 0).sum()) < 1700


@pytest.mark.parametrize("name", ["f32", "f64", "bf16"])
def test_dropout_of_nearly_all(nxv, torch, name):
    """p above the largest uniform, 1 - 2^-24, keeps nothing."""
    x = torch.full((5000,), 1.5, device="cuda", dtype=dt(torch, name))
    for p in (1 - 2.0 ** -24, 1 - 2.0 ** -25, 1 - 2.0 ** -53, 1.0):
        y = torch.full_like(x, 3.0)
        ok(nxv.dropout(wrap(nxv, x), p, 7, dtype=name, out=wrap(nxv, y)))
        # the first keeps the uniform 1 - 2^-24 alone, which these 5000 do not hold
        assert bool((y == 0).all())


def test_dropout_of_nothing(nxv, torch):
    ok(nxv.dropout(ok(nxv.upload_binary(b"")), 0.5, 1))


# ---- linear cross entropy ----------------------------------------------------------

# up to 2^26 multiply-adds (bf16 2^23) on one path, more on the tensor cores
XENT_SHAPES = [(1, 1, 1), (1, 10, 3), (3, 257, 13), (2, 256, 64), (130, 1000, 64), (129, 513, 65),
               (128, 256, 128), (257, 300, 1001), (5, 5003, 16), (300, 31, 200), (4099, 21, 17), (1, 70001, 5),
               (515, 515, 515), (513, 1001, 513), (129, 2049, 1025), (100, 40000, 64), (20000, 129, 64),
               (3001, 100, 1000), (3, 20000, 3000), (2, 50001, 700), (8193, 12, 800), (40000, 300, 8), (9000, 70, 130),
               (129, 600, 72), (200, 1100, 333),
               # up to 8 rows, with x in shared memory or (the last two) not
               (1, 31, 2048), (8, 1000, 2048), (7, 30000, 1024), (1, 100003, 640), (6, 9999, 41), (4, 5000, 4096), (8, 33, 8),
               (3, 1, 100), (2, 65536, 1000), (8, 700, 2056), (1, 500, 16392),
               (9, 65536, 64), (17, 30001, 100), (24, 2048, 2048), (16, 30000, 100), (12, 10001, 333), (13, 2000, 1000)]


def xent_inputs(torch, name, n, v, d, seed=0, scale=2.0):
    torch.manual_seed(seed + n * 7 + v * 3 + d)
    t = dt(torch, name)
    x = torch.randn(n, d, device="cuda").to(t)
    w = (torch.randn(v, d, device="cuda") * scale / d ** 0.5).to(t)
    labels = torch.randint(-1, v + 1, (n,), device="cuda")  # -1 and v: no target
    return x, w, labels


def xent_run(nxv, torch, x, w, labels, name, workspace=None, outs=None):
    n, d = x.shape
    loss, lse = outs or (torch.full((n,), 9.0, device="cuda"), torch.full((n,), 9.0, device="cuda"))
    ok(nxv.linear_cross_entropy(wrap(nxv, x), wrap(nxv, w), wrap(nxv, labels), n, w.shape[0], d,
                                dtype=name, index_bytes=labels.element_size(),
                                out=(wrap(nxv, loss), wrap(nxv, lse)), workspace=workspace))
    return loss, lse


def logit_tol(x, w, name):
    """Per row: the largest logit's possible error."""
    d = x.shape[1]
    # small problems: f32 FMAs in two or four strands, d / 2 roundings of 2^-24
    adds = d / 4 + 8 if name == "bf16" else 6 * (d / 16 + 1) + 8
    return (adds * 2.0 ** -23) * (x.double().abs() @ w.double().abs().t()).amax(1)


def lse_tol(z, ez):
    # every exponential: 2^-22, and 2^-23 of its exponent's size; log and sums: 2^-21 of their size
    return ez + 2.0 ** -20 * (4 + z.abs().amax(1) + np.log(z.shape[1]))


def xent_check(torch, name, x, w, labels, loss, lse):
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, 1)
    has = (labels >= 0) & (labels < w.shape[0])
    zl = z.gather(1, labels.long().clamp(0, w.shape[0] - 1)[:, None])[:, 0]
    ez = logit_tol(x, w, name)
    tol = lse_tol(z, ez)
    within(torch, lse, want, tol)
    within(torch, loss, torch.where(has, want - zl, 0.0), torch.where(has, tol + ez, 0.0))


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shape", XENT_SHAPES, ids=str)
def test_linear_cross_entropy(nxv, torch, name, shape):
    a = xent_inputs(torch, name, *shape)
    out = xent_run(nxv, torch, *a, name)
    xent_check(torch, name, *a, *out)
    again = xent_run(nxv, torch, *a, name)
    assert all(torch.equal(p, q) for p, q in zip(out, again))


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_linear_cross_entropy_int32_labels(nxv, torch, name):
    x, w, labels = xent_inputs(torch, name, 200, 77, 40)
    want = xent_run(nxv, torch, x, w, labels, name)
    got = xent_run(nxv, torch, x, w, labels.int(), name)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [1, 4])
def test_linear_cross_entropy_at_any_address(nxv, torch, name, shift):
    x, w, labels = xent_inputs(torch, name, 70, 300, 64)
    a = (place(torch, x, shift)[0], place(torch, w, shift)[0], labels)
    xent_check(torch, name, *a, *xent_run(nxv, torch, *a, name))


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_linear_cross_entropy_far_labels(nxv, torch, name):
    """Labels near the ends of 64 bits, and in 32 bits those whose low word is a class."""
    x, w, _ = xent_inputs(torch, name, 6, 40, 24)
    far = torch.tensor([-2 ** 63, 2 ** 63 - 1, 2 ** 32 + 3, -2 ** 32 + 3, 3, 39], device="cuda")
    loss, lse = xent_run(nxv, torch, x, w, far, name)
    assert loss[:4].tolist() == [0.0] * 4
    xent_check(torch, name, x, w, far, loss, lse)


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_linear_cross_entropy_large_logits(nxv, torch, name):
    """Logits of thousands: no overflow, and a loss near 0 where the label wins."""
    x, w, labels = xent_inputs(torch, name, 64, 600, 96, scale=2000.0)
    labels[:32] = (x[:32].double() @ w.double().t()).argmax(1)
    xent_check(torch, name, x, w, labels, *xent_run(nxv, torch, x, w, labels, name))


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_linear_cross_entropy_bad_rows_stay_their_own(nxv, torch, name):
    x, w, labels = xent_inputs(torch, name, 40, 300, 32)
    x[3, 5] = float("nan")
    x[17, 0] = float("inf")
    loss, lse = xent_run(nxv, torch, x, w, labels, name)
    assert bool(torch.isnan(lse[[3, 17]]).all())
    keep = [i for i in range(40) if i not in (3, 17)]
    xent_check(torch, name, x[keep], w, labels[keep], loss[keep], lse[keep])


def test_linear_cross_entropy_class_of_minus_infinity_bf16(nxv, torch):
    """A class whose logits are -inf takes no part; a row with only such classes has lse NaN."""
    x, w, labels = xent_inputs(torch, "bf16", 20, 50, 16)
    x = x.abs() + 0.25
    w[7] = float("-inf")
    labels[:] = 3
    loss, lse = xent_run(nxv, torch, x, w, labels, "bf16")
    rest = [v for v in range(50) if v != 7]
    xent_check(torch, "bf16", x, w[rest], labels, loss, lse)
    w[:] = float("-inf")
    assert bool(torch.isnan(xent_run(nxv, torch, x, w, labels, "bf16")[1]).all())


def xgrad_run(nxv, torch, dl, x, w, labels, lse, name, workspace=None, outs=None):
    n, d = x.shape
    dx, dw = outs or (torch.full_like(x, 9.0), torch.full_like(w, 9.0))
    ok(nxv.linear_cross_entropy_grad(*(wrap(nxv, t) for t in (dl, x, w, labels, lse)), n, w.shape[0], d,
                                     dtype=name, index_bytes=labels.element_size(),
                                     out=(wrap(nxv, dx), wrap(nxv, dw)), workspace=workspace))
    return dx, dw


def xgrad_check(torch, name, dl, x, w, labels, lse, dx, dw):
    n, v = x.shape[0], w.shape[0]
    has = (labels >= 0) & (labels < v)
    X, W = torch.where(has[:, None], x.double(), 0.0), w.double()
    z = X @ W.t()
    p = torch.exp(z - lse.double()[:, None])
    hot = torch.zeros_like(p)
    hot[has, labels[has].long()] = 1.0
    DL = torch.where(has, dl.double(), 0.0)[:, None]
    g = (p - hot) * DL
    # p: the logit's error, 2^-21 and 2^-22 of the exponent; the difference with 1 rounds once more
    ez = logit_tol(X, w, name)[:, None]
    eg = DL.abs() * (p * (1.01 * ez + 2.0 ** -21 + 2.0 ** -22 * (z - lse.double()[:, None]).abs()) + hot * 2.0 ** -23)
    hg = 2.0 ** -8 if name == "bf16" else 2.0 ** -23
    six = 1 if name == "bf16" else 6
    eg = eg + hg * (g.abs() + eg)
    gm = g.abs() + eg
    want = g @ W
    # K = v classes in pieces, each joined with one more addition
    within(torch, dx, want, H[name] * want.abs() + eg @ W.abs()
           + (max(six * (v / 16 + 1), v / 4) + 8 + v / 1024) * 2.0 ** -23 * (gm @ W.abs()))
    want = g.t() @ X
    # dloss x is rounded too, to the type of the products: one more half step of each term
    within(torch, dw, want, H[name] * want.abs() + (eg + hg * gm).t() @ X.abs()
           + (max(six * (n / 16 + 1), n / 4) + 8) * 2.0 ** -23 * (gm.t() @ X.abs()))


def xgrad_inputs(torch, name, n, v, d, seed=0):
    x, w, labels = xent_inputs(torch, name, n, v, d, seed)
    lse = torch.logsumexp(x.double() @ w.double().t(), 1).float()
    return torch.randn(n, device="cuda"), x, w, labels, lse


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shape", XENT_SHAPES, ids=str)
def test_linear_cross_entropy_grad(nxv, torch, name, shape):
    a = xgrad_inputs(torch, name, *shape)
    out = xgrad_run(nxv, torch, *a, name)
    xgrad_check(torch, name, *a, *out)
    again = xgrad_run(nxv, torch, *a, name)
    assert all(torch.equal(p, q) for p, q in zip(out, again))


@pytest.mark.parametrize("name,n,v,d", [("bf16", 3001, 70001, 72), ("f32", 3001, 30011, 36)])
def test_linear_cross_entropy_grad_in_pieces(nxv, torch, name, n, v, d):
    """More classes than one piece of the vocabulary."""
    a = xgrad_inputs(torch, name, n, v, d)
    xgrad_check(torch, name, *a, *xgrad_run(nxv, torch, *a, name))
    xent_check(torch, name, *a[1:4], *xent_run(nxv, torch, *a[1:4], name))


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [1, 4])
def test_linear_cross_entropy_grad_at_any_address(nxv, torch, name, shift):
    dl, x, w, labels, lse = xgrad_inputs(torch, name, 70, 300, 64)
    x, w = place(torch, x, shift)[0], place(torch, w, shift)[0]
    dx, r1 = place(torch, torch.zeros_like(x), shift)
    dw, r2 = place(torch, torch.zeros_like(w), shift)
    xgrad_run(nxv, torch, dl, x, w, labels, lse, name, outs=(dx, dw))
    xgrad_check(torch, name, dl, x, w, labels, lse, dx, dw)
    for r, t in ((r1, x), (r2, w)):
        assert bool((r[:shift] == 7).all()) and bool((r[shift + t.numel():] == 7).all())


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_rows_without_a_target_give_nothing(nxv, torch, name):
    """Whatever they hold: NaN and infinities in x, in their lse and in their incoming gradient."""
    dl, x, w, labels, lse = xgrad_inputs(torch, name, 150, 300, 48)
    labels[10:30] = -1
    labels[140:] = 300
    clean = xgrad_run(nxv, torch, dl, x, w, labels, lse, name)
    x, dl, lse = x.clone(), dl.clone(), lse.clone()
    x[10:20], x[20:30] = float("nan"), float("inf")
    dl[10:30], lse[10:30] = float("nan"), float("nan")
    got = xgrad_run(nxv, torch, dl, x, w, labels, lse, name)
    assert all(torch.equal(p, q) for p, q in zip(got, clean))
    assert bool((got[0][10:30] == 0).all()) and bool((got[0][140:] == 0).all())
    labels[:] = -1
    dx, dw = xgrad_run(nxv, torch, dl, x, w, labels, lse, name)
    assert bool((dx == 0).all()) and bool((dw == 0).all())


def test_linear_cross_entropy_past_32_bits(nxv, torch):
    """Weights of more than 2^31 elements, classes behind them as labels."""
    n, v, d = 130, (1 << 18) + 77, 8200
    torch.manual_seed(3)
    x = torch.randn(n, d, device="cuda").bfloat16()
    w = torch.empty(v, d, device="cuda", dtype=torch.bfloat16).normal_() * (2 / d ** 0.5)
    labels = torch.randint(v - 100, v, (n,), device="cuda")
    labels[0], labels[1] = 0, -1
    loss, lse = xent_run(nxv, torch, x, w, labels, "bf16")
    z = torch.cat([x.double() @ w[i:i + 4096].double().t() for i in range(0, v, 4096)], 1)
    want = torch.logsumexp(z, 1)
    # a logit's additions, at the largest size of a row's products
    size = [(x.double().abs() @ w[i:i + 4096].double().abs().t()).amax(1) for i in range(0, v, 4096)]
    ez = (d / 4 + 8) * 2.0 ** -23 * torch.stack(size).amax(0)
    tol = lse_tol(z, ez)
    within(torch, lse, want, tol)
    has = labels >= 0
    within(torch, loss[has], (want - z.gather(1, labels.clamp(min=0)[:, None])[:, 0])[has], (tol + ez)[has])
    dl = torch.full((n,), 1 / 129, device="cuda")
    dx, dw = xgrad_run(nxv, torch, dl, x, w, labels, lse, "bf16")
    p = torch.exp(z - lse.double()[:, None])
    p[has, labels[has]] -= 1.0
    g = torch.where(has[:, None], p * dl.double()[:, None], 0.0)
    for part in (slice(0, 50), slice(v - 120, v)):
        want = g[:, part].t() @ x.double()
        size = g[:, part].abs().t() @ x.double().abs()
        # two roundings to bf16 of every term and one of the sum; the logits' error
        within(torch, dw[part], want, 2.0 ** -8 * want.abs() + (2.0 ** -7 + 2 * float(ez.max()) + 2.0 ** -12) * size)
    want = torch.zeros(n, d, device="cuda", dtype=torch.float64)
    size = torch.zeros_like(want)
    for i in range(0, v, 4096):
        want += g[:, i:i + 4096] @ w[i:i + 4096].double()
        size += g[:, i:i + 4096].abs() @ w[i:i + 4096].double().abs()
    within(torch, dx, want, 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * float(ez.max()) + 2.0 ** -12 + v / 16 * 2.0 ** -23) * size)


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_no_rows(nxv, torch, name):
    x = torch.empty(0, 8, device="cuda", dtype=dt(torch, name))
    w = torch.randn(20, 8, device="cuda").to(x.dtype)
    e, l = torch.empty(0, device="cuda"), torch.empty(0, device="cuda", dtype=torch.int64)
    xent_run(nxv, torch, x, w, l, name)
    _, dw = xgrad_run(nxv, torch, e, x, w, l, e, name)
    assert bool((dw == 0).all())


def test_linear_cross_entropy_grad_against_differences(nxv, torch):
    """Along a random direction of (x, w), in f32: the losses of 40 rows are off by about 2^-21 each, so a
    difference over 2 h = 2^-5 by 40 * 2^-21 * 2^5 = 6e-4, and h^2 / 6 = 4e-5 times a third derivative of about 1 a row."""
    x, w, labels = xent_inputs(torch, "f32", 40, 70, 30)
    loss, lse = xent_run(nxv, torch, x, w, labels, "f32")
    one = torch.ones(40, device="cuda")
    dx, dw = xgrad_run(nxv, torch, one, x, w, labels, lse, "f32")
    ex, ew = torch.randn_like(x) / 30 ** 0.5, torch.randn_like(w) / 30 ** 0.5
    h = 2.0 ** -6
    f = lambda t: xent_run(nxv, torch, x + t * ex, w + t * ew, labels, "f32")[0].double().sum()  # noqa: E731
    want = float((f(h) - f(-h)) / (2 * h))
    got = float((dx.double() * ex).sum() + (dw.double() * ew).sum())
    assert abs(got - want) <= 6e-4 + 40 * 4e-5 * 4


# ---- together -----------------------------------------------------------------------

def test_the_end_of_a_network(nxv, torch):
    """norm -> dropout -> cross entropy and back through all three, f32, against autograd in 64 bits.

    Relative 2-norms.  The products' worst case for dim 96: (6 * 7 + 8) 2^-23 = 6e-6 each, of which a
    gradient passes two in a row (the logits and its own), 1.2e-5; the norm's 128 * 2^-24 = 8e-6 in each direction: 2.8e-5."""
    n, v, d, p, seed = 200, 777, 96, 0.2, 99
    torch.manual_seed(5)
    x = torch.randn(n, d, device="cuda") * 2 + 0.3
    g, b = torch.randn(d, device="cuda") * 0.2 + 1, torch.randn(d, device="cuda") * 0.2
    w = torch.randn(v, d, device="cuda") * 2 / d ** 0.5
    labels = torch.randint(-1, v, (n,), device="cuda")
    y, m, s = norm_run(nxv, torch, x, g, b, 1e-5, "f32")
    h = torch.empty_like(y)
    ok(nxv.dropout(wrap(nxv, y), p, seed, out=wrap(nxv, h)))
    loss, lse = xent_run(nxv, torch, h, w, labels, "f32")
    has = labels >= 0
    dl = torch.full((n,), 1.0, device="cuda") / has.sum()
    dh, dw = xgrad_run(nxv, torch, dl, h, w, labels, lse, "f32")
    ok(nxv.dropout(wrap(nxv, dh), p, seed, out=wrap(nxv, dh)))
    dx, dg, db = grad_run(nxv, torch, dh, x, g, m, s, "f32")

    X, G, B, W = (t.double().requires_grad_() for t in (x, g, b, w))
    M = X.mean(1, keepdim=True)
    Y = (X - M) / ((X - M).square().mean(1, keepdim=True) + 1e-5).sqrt() * G + B
    keep = torch.from_numpy(mask_of(nxv, seed, 0, n * d, p)).cuda().view(n, d)
    Z = torch.where(keep, Y / (1 - p), 0.0) @ W.t()
    L = torch.logsumexp(Z, 1) - Z.gather(1, labels.clamp(min=0)[:, None])[:, 0]
    (L[has].sum() / has.sum()).backward()
    within(torch, loss[has], L[has].detach(), 2.8e-5 * (1 + Z.detach().abs().amax(1)[has]))
    assert bool((loss[~has] == 0).all())
    for got, want in ((dx, X.grad), (dg, G.grad), (db, B.grad), (dw, W.grad)):
        assert float((got.double() - want).norm() / want.norm()) <= 2.8e-5


def test_on_another_stream(nxv, torch):
    from nx_vulkan_b200 import _native
    a = xgrad_inputs(torch, "bf16", 200, 500, 64)
    want = xgrad_run(nxv, torch, *a, "bf16")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    _native.load().nxv_set_stream(side.cuda_stream)
    with torch.cuda.stream(side):
        got = xgrad_run(nxv, torch, *a, "bf16")
        side.synchronize()
    _native.load().nxv_set_stream(1)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_captured_and_replayed(nxv, torch):
    """Two graphs with a workspace each, replayed at the same time on two streams with new inputs."""
    from nx_vulkan_b200 import _native
    lib = _native.load()
    n, v, d = 150, 700, 64
    sets = []
    for i in range(2):
        dl, x, w, labels, lse = xgrad_inputs(torch, "bf16", n, v, d, seed=i)
        g, m = x[0].clone(), torch.empty(n, device="cuda")
        st = {"in": (x, w, labels), "dl": dl, "gamma": g, "mean": m, "rstd": torch.empty_like(m),
              "y": torch.empty_like(x), "h": torch.empty_like(x), "loss": torch.empty_like(m),
              "lse": torch.empty_like(m), "dx": torch.empty_like(x), "dw": torch.empty_like(w),
              "dg": torch.empty_like(g), "db": torch.empty_like(g), "dn": torch.empty_like(x)}
        need = max(nxv.linear_cross_entropy_workspace(n, v, d, "bf16"),
                   nxv.linear_cross_entropy_workspace(n, v, d, "bf16", grad=True),
                   nxv.layer_norm_grad_workspace(n, d, "bf16"))
        st["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        st["wsh"] = wrap(nxv, st["ws"])
        sets.append(st)

    def step(st, ws):
        x, w, labels = st["in"]
        h = lambda k: wrap(nxv, st[k])  # noqa: E731
        ok(nxv.layer_norm(wrap(nxv, x), h("gamma"), h("gamma"), n, d, dtype="bf16", out=(h("y"), h("mean"), h("rstd"))))
        ok(nxv.dropout(h("y"), 0.1, 7, dtype="bf16", out=h("h")))
        xent_run(nxv, torch, st["h"], w, labels, "bf16", workspace=ws, outs=(st["loss"], st["lse"]))
        xgrad_run(nxv, torch, st["dl"], st["h"], w, labels, st["lse"], "bf16", workspace=ws, outs=(st["dx"], st["dw"]))
        ok(nxv.dropout(h("dx"), 0.1, 7, dtype="bf16", out=h("dx")))
        ok(nxv.layer_norm_grad(h("dx"), wrap(nxv, x), h("gamma"), h("mean"), h("rstd"), n, d, dtype="bf16",
                               out=(h("dn"), h("dg"), h("db")), workspace=ws))

    keys = ("y", "mean", "rstd", "loss", "lse", "dx", "dw", "dn", "dg", "db")
    graphs, streams = [], [torch.cuda.Stream() for _ in sets]
    for st, s in zip(sets, streams):
        step(st, st["wsh"])
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            lib.nxv_set_stream(s.cuda_stream)
            step(st, st["wsh"])
        lib.nxv_set_stream(1)
        graphs.append(gr)
    fresh = [xent_inputs(torch, "bf16", n, v, d, seed=10 + i) for i in range(2)]
    for st, f in zip(sets, fresh):
        for t, u in zip(st["in"], f):
            t.copy_(u)
    torch.cuda.synchronize()
    for _ in range(3):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    got = [{k: st[k].clone() for k in keys} for st in sets]
    for st, g in zip(sets, got):
        for k in keys:
            st[k].fill_(5.0)
        step(st, None)
        torch.cuda.synchronize()
        for k in keys:
            assert torch.equal(st[k], g[k]), k
    del graphs


def test_a_capture_needs_its_own_workspace(nxv, torch):
    from nx_vulkan_b200 import _native
    lib = _native.load()
    dl, x, w, labels, lse = xgrad_inputs(torch, "bf16", 20, 30, 16)
    dx, dw, loss = torch.empty_like(x), torch.empty_like(w), torch.empty(20, device="cuda")
    hs = [wrap(nxv, t) for t in (dl, x, w, labels, lse, dx, dw, loss)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=s):
        lib.nxv_set_stream(s.cuda_stream)
        r = nxv.linear_cross_entropy_grad(*hs[:5], 20, 30, 16, dtype="bf16", out=(hs[5], hs[6]))
        said = _native.last_error()
        q = nxv.linear_cross_entropy(hs[1], hs[2], hs[3], 20, 30, 16, dtype="bf16", out=(hs[7], hs[4]))
        k = nxv.layer_norm_grad(hs[1], hs[1], hs[1], hs[4], hs[4], 20, 16, dtype="bf16", out=(hs[5], hs[6], hs[7]))
        # ... and its own outputs
        o = [nxv.dropout(hs[1], 0.5, 1), nxv.linear_cross_entropy(hs[1], hs[2], hs[3], 20, 30, 16, dtype="bf16")]
        lib.nxv_set_stream(1)
        loss.zero_()  # the graph is not empty
    assert o[0] == o[1] == ("error", "alloc_failed")
    assert r == ("error", "dispatch_failed") and "workspace" in said
    assert q == ("error", "dispatch_failed") and k[0] == "error"


def test_refusals_on_device(nxv, torch):
    from nx_vulkan_b200 import _native
    lib = _native.load()
    big = torch.zeros(4096, device="cuda")
    kept = []  # handles live until the end of the test

    def W(a, n):
        kept.append(nxv.wrap_tensor(big[a:a + n]))
        return kept[-1]

    x, y, v = W(0, 64), W(1024, 64), W(2048, 16)
    st = (W(2100, 4), W(2200, 4))

    def refused(rc, part):
        assert rc == -3 and part in _native.last_error(), (rc, _native.last_error())

    ln = lambda y, x: lib.nxv_layer_norm(y.handle, st[0].handle, st[1].handle, x.handle, v.handle,  # noqa: E731
                                         v.handle, 4, 16, 1e-5, 0, b"layer_norm.spv")
    assert ln(y, x) == 0 and ln(x, x) == 0
    refused(ln(W(4, 64), x), "shares memory")          # overlaps x without being x
    refused(ln(W(1024, 60), x), "needs 256")           # too small
    refused(ln(W(2100, 64), x), "shares memory")       # over the statistics
    odd = lib.nxv_buf_wrap(C.c_void_p(big.data_ptr() + 2), 64 * 4)
    rc = lib.nxv_layer_norm(odd, st[0].handle, st[1].handle, x.handle, v.handle, v.handle, 4, 16,
                            1e-5, 0, b"layer_norm.spv")
    refused(rc, "not a multiple")
    lib.nxv_buf_free(odd)
    lg = lambda dx, dg, ws: lib.nxv_layer_norm_grad(dx.handle, dg.handle, W(2500, 16).handle, ws, y.handle,  # noqa: E731
                                                    x.handle, v.handle, st[0].handle, st[1].handle, 4, 16, 0,
                                                    b"layer_norm_grad.spv")
    need = nxv.layer_norm_grad_workspace(4, 16) // 4
    dx, dg, ws = W(256, 64), W(2400, 16), W(2560, need)
    assert lg(dx, dg, None) == 0 and lg(dx, dg, ws.handle) == 0 and lg(y, dg, ws.handle) == 0
    refused(lg(W(1028, 64), dg, None), "shares memory")
    refused(lg(dx, v, None), "shares memory")
    refused(lg(dx, dg, W(2560, need - 1).handle), "workspace")
    refused(lg(dx, dg, W(2562, need).handle), "workspace")
    refused(lg(dx, dg, W(0, need).handle), "shares memory")
    dr = lambda o, x: lib.nxv_dropout(o.handle, x.handle, 64, 0.5, 1, 0, 0, b"dropout.spv")  # noqa: E731
    assert dr(y, x) == 0 and dr(x, x) == 0
    refused(dr(W(1, 64), x), "shares memory")
    refused(dr(W(1024, 63), x), "needs 256")
    lab = nxv.wrap_tensor(big[3000:3008])  # four labels of 0
    ce = lambda loss, lse: lib.nxv_linear_cross_entropy(loss.handle, lse.handle, None, x.handle, y.handle,  # noqa: E731
                                                        lab.handle, 4, 4, 16, 0, 8,
                                                        b"linear_cross_entropy.spv")
    assert ce(*st) == 0
    refused(ce(st[0], st[0]), "shares memory")
    refused(ce(W(10, 4), st[0]), "shares memory")
    cg = lambda dx, dw: lib.nxv_linear_cross_entropy_grad(dx.handle, dw.handle, None, st[0].handle, x.handle,  # noqa: E731
                                                          y.handle, lab.handle, st[1].handle, 4, 4,
                                                          16, 0, 8, b"linear_cross_entropy_grad.spv")
    assert cg(W(256, 64), W(400, 64)) == 0
    refused(cg(x, W(400, 64)), "shares memory")
    refused(cg(W(256, 64), y), "shares memory")
    refused(cg(W(256, 64), W(300, 64)), "shares memory")
    torch.cuda.synchronize()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(3, 300, 48), (1, 1000, 333), (8, 2000, 77), (12, 30000, 100), (40, 300, 48), (200, 900, 70)],
                         ids=str)
def test_every_path_with_a_row_of_nan_int32_labels_and_a_replay(nxv, torch, name, shape):
    """A workspace of just the stated size, kept to; a row without a target that holds NaN."""
    from nx_vulkan_b200 import _native
    n, v, d = shape
    dl, x, w, labels, lse = xgrad_inputs(torch, name, n, v, d)
    row = n // 2
    labels[row] = -1
    rooms, sized = [], []
    for grad in (False, True):
        need = nxv.linear_cross_entropy_workspace(n, v, d, name, grad=grad)
        rooms.append(torch.full((need + 4096,), 77, dtype=torch.uint8, device="cuda"))
        sized.append((need, wrap(nxv, rooms[-1][:need])))
    want = [t.clone() for t in xgrad_run(nxv, torch, dl, x, w, labels, lse, name)]
    loss = xent_run(nxv, torch, x, w, labels, name)[0].clone()
    x[row], dl[row], lse[row] = float("nan"), float("nan"), float("nan")
    labels = labels.int()
    outs = [torch.full_like(loss, 9.0), torch.full_like(loss, 9.0)], [torch.full_like(x, 9.0), torch.full_like(w, 9.0)]

    def both():
        xent_run(nxv, torch, x, w, labels, name, workspace=sized[0][1], outs=outs[0])
        xgrad_run(nxv, torch, dl, x, w, labels, lse, name, workspace=sized[1][1], outs=outs[1])

    both()
    torch.cuda.synchronize()
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=s):
        _native.load().nxv_set_stream(s.cuda_stream)
        both()
    _native.load().nxv_set_stream(1)
    for replay in (False, True):
        if replay:
            for t in (*outs[0], *outs[1]):
                t.fill_(9.0)
            graph.replay()
            torch.cuda.synchronize()
        rest = torch.arange(n, device="cuda") != row
        assert torch.equal(outs[0][0][rest], loss[rest]) and float(outs[0][0][row]) == 0.0
        assert all(torch.equal(p, q) for p, q in zip(outs[1], want))
    for room, (need, _) in zip(rooms, sized):
        assert bool((room[need:] == 77).all())
