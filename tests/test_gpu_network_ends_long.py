"""Layer norm of rows that are longer than any sum in f32 can be, up to the limit of 2^28 columns.

Tolerances.  u = 2^-24 (f64 2^-53), h as in test_gpu_network_ends.py.  Sums along the row lose nothing that counts
(f64: 2^18 additions of 2^-53 at most), so the mean is off by its own rounding, u |mean|; a centred value by that and a
rounding; rstd by 4 roundings and the square of the mean's error; y by 4 more.  In the gradient a thread adds 16 values
of a lane in f32 before they join its f64 sums: with the products' roundings and the formula's own, 32 u."""
import pytest

from test_gpu_network_ends import H, U, _stream, dt, grad_run, norm_run, stat, torch, within  # noqa: F401

pytestmark = pytest.mark.gpu


def row(torch, name, cols):
    torch.manual_seed(cols)
    x = torch.empty(1, cols, device="cuda", dtype=torch.float32).normal_().add_(1003.3)
    return x.to(dt(torch, name))


@pytest.mark.parametrize("name,cols", [("f32", 1 << 26), ("f32", 1 << 28), ("bf16", 1 << 28), ("bf16", (1 << 26) + 5),
                                       ("f32", 70001), ("f64", 1 << 26), ("f64", 40001)])
def test_layer_norm_of_a_long_row(nxv, torch, name, cols):
    x = row(torch, name, cols)
    g = torch.empty(cols, device="cuda").normal_().to(x.dtype)
    b = torch.empty(cols, device="cuda").normal_().to(x.dtype)
    y, m, s = norm_run(nxv, torch, x, g, b, 1e-5, name)
    u, X = U[name], x.double()
    # torch's own sums of 2^28 f64 values: 28 levels and some in turn, below u for f32; twice u allowed for f64
    M = X.mean(1, keepdim=True)
    S = 1 / ((X - M).square().mean(1, keepdim=True) + 1e-5).sqrt()
    more = 64 * u if name == "f64" else 0.0  # here 2^18 / 2 sequential f64 additions of a thread, random in sign
    size = M.abs()
    within(torch, m[:, None], M, (2 * u + more) * size)
    within(torch, s[:, None], S, S * (8 * u + more + ((2 * u + more) * size * S) ** 2))
    del X
    bad = 0
    for a in range(0, cols, 1 << 25):
        p = slice(a, a + (1 << 25))
        xh = (x[0, p].double() - M[0]) * S[0]
        G, B = g[p].double(), b[p].double()
        want = xh * G + B
        k = (8 * u + more) * (G.abs() * (xh.abs() + size[0] * S[0]) + B.abs())
        bad += int(((y[0, p].double() - want).abs() > H[name] * want.abs() + k).sum())
    assert bad == 0


@pytest.mark.parametrize("name,cols", [("f32", 1 << 26), ("f32", (1 << 26) + 3), ("bf16", 1 << 27), ("f64", 1 << 25),
                                       ("f32", 40001)])
def test_layer_norm_grad_of_a_long_row(nxv, torch, name, cols):
    """The gradient of a mean: the same dy everywhere, whose sum in f32 drifts one way."""
    x = row(torch, name, cols)
    X = x.double()
    m = X.mean(1).to(stat(torch, name))
    s = (1 / ((X - m.double()[:, None]).square().mean(1) + 1e-5).sqrt()).to(stat(torch, name))
    dy, g = torch.full_like(x, 0.3), torch.full((cols,), 1.0, device="cuda", dtype=x.dtype)
    dx, dg, db = grad_run(nxv, torch, dy, x, g, m, s, name)
    u, M, S = U[name], m.double(), s.double()
    w = float(dy[0, 0])
    xh = (X[0] - M) * S
    a, q, aq = w, float((w * xh).mean()), float((w * xh).abs().mean())
    want = S * (w - a - xh * q)
    k = 32 * u + (2 ** 16 * u if name == "f64" else 0.0)  # f64: its own sequential additions
    within(torch, dx[0], want, H[name] * want.abs() + k * S * (2 * w + xh.abs() * aq))
    within(torch, dg, w * xh, (H[name] + 4 * u) * (w * xh).abs() + 4 * u * w * S * M.abs())
    assert bool((db == dy[0]).all())
