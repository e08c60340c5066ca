"""The linear cross entropy's special cases at sizes that the tensor cores take: labels, addresses, rows without a
target, NaN and infinities, streams, captured graphs, host threads.

Tolerances are those of test_gpu_network_ends.py; what has one arithmetic has to be equal bit for bit."""
import threading

import pytest

from test_gpu_network_ends import (_stream, dt, norm_run, ok, place, torch, within, wrap, xent_check,  # noqa: F401
                                   xent_inputs, xent_run, xgrad_check, xgrad_inputs, xgrad_run)

pytestmark = pytest.mark.gpu

TYPES = ["f32", "bf16"]
# single CTAs' tiles, dx in slices of the classes; pairs' tiles; dw in slices of the rows, rows that are no whole
# 16-byte pieces in bf16
SHAPES = [(300, 2000, 96), (2100, 2100, 72), (5000, 200, 70)]


def on_tensor_cores(nxv, n, v, d, name):
    """Only there the forward workspace has room for packed x and w (and few rows go elsewhere)."""
    planes, dp = (3 if name == "f32" else 1), (d + 63) // 64 * 64
    return n > 24 and nxv.linear_cross_entropy_workspace(n, v, d, name) >= planes * 2 * (n + v) * dp


@pytest.fixture(params=SHAPES, ids=str)
def shape(request):
    return request.param


@pytest.mark.parametrize("name", TYPES)
def test_these_sizes_are_the_tensor_cores(nxv, shape, name):
    assert on_tensor_cores(nxv, *shape, name)
    assert not on_tensor_cores(nxv, 64, 100, 50, name) and not on_tensor_cores(nxv, 4, 70000, 96, name)


@pytest.mark.parametrize("name", TYPES)
def test_int32_labels(nxv, torch, shape, name):
    dl, x, w, labels, lse = xgrad_inputs(torch, name, *shape)
    for run, a in ((xent_run, (x, w)), (xgrad_run, (dl, x, w))):
        more = () if run is xent_run else (lse,)
        want = run(nxv, torch, *a, labels, *more, name)
        got = run(nxv, torch, *a, labels.int(), *more, name)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shift", [1, 4])
def test_at_any_address(nxv, torch, shape, name, shift):
    dl, x, w, labels, lse = xgrad_inputs(torch, name, *shape)
    x, w = place(torch, x, shift)[0], place(torch, w, shift)[0]
    xent_check(torch, name, x, w, labels, *xent_run(nxv, torch, x, w, labels, name))
    dx, r1 = place(torch, torch.zeros_like(x), shift)
    dw, r2 = place(torch, torch.zeros_like(w), shift)
    xgrad_run(nxv, torch, dl, x, w, labels, lse, name, outs=(dx, dw))
    xgrad_check(torch, name, dl, x, w, labels, lse, dx, dw)
    for r, t in ((r1, x), (r2, w)):
        assert bool((r[:shift] == 7).all()) and bool((r[shift + t.numel():] == 7).all())


@pytest.mark.parametrize("name", TYPES)
def test_far_labels(nxv, torch, shape, name):
    """Labels near the ends of 64 bits, and those whose low 32 bits are a class, have no target."""
    dl, x, w, labels, lse = xgrad_inputs(torch, name, *shape)
    far = torch.tensor([-2 ** 63, 2 ** 63 - 1, 2 ** 32 + 3, -2 ** 32 + 3, -1, shape[1]], device="cuda")
    labels = torch.randint(0, shape[1], labels.shape, device="cuda")
    labels[10:16] = far
    loss, out = xent_run(nxv, torch, x, w, labels, name)
    assert loss[10:16].tolist() == [0.0] * 6
    xent_check(torch, name, x, w, labels, loss, out)
    dx, dw = xgrad_run(nxv, torch, dl, x, w, labels, lse, name)
    assert bool((dx[10:16] == 0).all())
    labels[10:16] = -1
    assert all(torch.equal(p, q) for p, q in zip(xgrad_run(nxv, torch, dl, x, w, labels, lse, name), (dx, dw)))


@pytest.mark.parametrize("name", TYPES)
def test_large_logits(nxv, torch, shape, name):
    """Logits of thousands: no overflow, and a loss near 0 where the label wins."""
    x, w, labels = xent_inputs(torch, name, *shape, scale=2000.0)
    labels[:100] = (x[:100].double() @ w.double().t()).argmax(1)
    xent_check(torch, name, x, w, labels, *xent_run(nxv, torch, x, w, labels, name))


@pytest.mark.parametrize("name", TYPES)
def test_loss_of_a_label_that_wins(nxv, torch, shape, name):
    """The label's logit is L, all others are 0: the loss, log(1 + (v - 1) e^-L), is not below 0 and off by what the
    terms and the logarithm are off, whatever L's size.  The largest term is exactly 1; the others are 2^-22 of
    themselves off and 2^-24 of their exponent's size, twice; sums round by 2^-24 for each of a thread's 32 columns and
    12 levels, but never below 1; logf is off by an ulp."""
    n, v, d = shape
    for L in (9.3125, 30.75, 50.125, 77.0, 101.25, 1003.0):
        L = float(torch.tensor(L, dtype=dt(torch, name)))  # what x holds
        x = torch.zeros(n, d, device="cuda", dtype=dt(torch, name))
        w = torch.zeros(v, d, device="cuda", dtype=dt(torch, name))
        labels = torch.arange(n, device="cuda") % min(v, d)
        x[torch.arange(n), labels] = L
        w[torch.arange(min(v, d)), torch.arange(min(v, d))] = 1.0
        loss, lse = xent_run(nxv, torch, x, w, labels, name)
        rest = (v - 1) * torch.exp(torch.tensor(-L, dtype=torch.float64))
        assert float(loss.min()) >= 0.0, (L, float(loss.min()))
        tol = float(rest) * (2.0 ** -22 + 2 * L * 2.0 ** -24) + 44 * 2.0 ** -24 * (1.0 if float(rest) > 2.0 ** -24 else 0.0)
        within(torch, loss, torch.log1p(rest).cuda().expand(n), tol + 2.0 ** -23)
        within(torch, lse, (L + torch.log1p(rest)).cuda().expand(n), tol + 2.0 ** -23 + L * 2.0 ** -24)


@pytest.mark.parametrize("name", TYPES)
def test_bad_rows_stay_their_own(nxv, torch, shape, name):
    x, w, labels = xent_inputs(torch, name, *shape)
    bad = [3, 17, 140]
    x[3, 5], x[17, 0], x[140] = float("nan"), float("inf"), float("-inf")
    loss, lse = xent_run(nxv, torch, x, w, labels, name)
    assert bool(torch.isnan(lse[bad]).all())
    keep = [i for i in range(shape[0]) if i not in bad]
    xent_check(torch, name, x[keep], w, labels[keep], loss[keep], lse[keep])


def test_class_of_minus_infinity_bf16(nxv, torch, shape):
    """A class whose logits are -inf takes no part; a row with only such classes has lse NaN."""
    x, w, labels = xent_inputs(torch, "bf16", *shape)
    x = x.abs() + 0.25
    w[7] = float("-inf")
    labels[:] = 3
    loss, lse = xent_run(nxv, torch, x, w, labels, "bf16")
    rest = [v for v in range(shape[1]) if v != 7]
    xent_check(torch, "bf16", x, w[rest], labels, loss, lse)
    w[:] = float("-inf")
    assert bool(torch.isnan(xent_run(nxv, torch, x, w, labels, "bf16")[1]).all())


@pytest.mark.parametrize("name", TYPES)
def test_rows_without_a_target_give_nothing(nxv, torch, shape, name):
    """Whatever they hold: NaN and infinities in x, in their lse and in their incoming gradient."""
    dl, x, w, labels, lse = xgrad_inputs(torch, name, *shape)
    labels[10:30] = -1
    labels[140:150] = shape[1]
    clean = xgrad_run(nxv, torch, dl, x, w, labels, lse, name)
    x, dl, lse = x.clone(), dl.clone(), lse.clone()
    x[10:20], x[20:30] = float("nan"), float("inf")
    dl[10:30], lse[10:30] = float("nan"), float("nan")
    got = xgrad_run(nxv, torch, dl, x, w, labels, lse, name)
    assert all(torch.equal(p, q) for p, q in zip(got, clean))
    assert bool((got[0][10:30] == 0).all()) and bool((got[0][140:150] == 0).all())
    labels[:] = -1
    dx, dw = xgrad_run(nxv, torch, dl, x, w, labels, lse, name)
    assert bool((dx == 0).all()) and bool((dw == 0).all())


def workspaces(nxv, torch, n, v, d, name):
    """Of just the stated size, with what lies behind them."""
    rooms, sized = [], []
    for grad in (False, True):
        need = nxv.linear_cross_entropy_workspace(n, v, d, name, grad=grad)
        rooms.append(torch.full((need + 4096,), 77, dtype=torch.uint8, device="cuda"))
        sized.append(wrap(nxv, rooms[-1][:need]))
    return rooms, sized, [r.numel() - 4096 for r in rooms]


@pytest.mark.parametrize("name", TYPES)
def test_two_graphs_at_once(nxv, torch, shape, name):
    """Each with workspaces of its own, of just the stated size and kept to; replayed at the same time on two
    streams with new inputs, one row of them without a target and full of NaN."""
    from nx_vulkan_b200 import _native
    lib = _native.load()
    sets = []
    for i in range(2):
        dl, x, w, labels, _ = xgrad_inputs(torch, name, *shape, seed=i)
        n = shape[0]
        sets.append({"in": (dl, x, w, labels.int()), "lse": torch.empty(n, device="cuda"),
                     "loss": torch.empty(n, device="cuda"), "dx": torch.empty_like(x), "dw": torch.empty_like(w),
                     "ws": workspaces(nxv, torch, *shape, name)})

    def step(st, ws):
        dl, x, w, labels = st["in"]
        xent_run(nxv, torch, x, w, labels, name, workspace=ws[0], outs=(st["loss"], st["lse"]))
        xgrad_run(nxv, torch, dl, x, w, labels, st["lse"], name, workspace=ws[1], outs=(st["dx"], st["dw"]))

    graphs, streams = [], [torch.cuda.Stream() for _ in sets]
    for st, s in zip(sets, streams):
        step(st, st["ws"][1])
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            lib.nxv_set_stream(s.cuda_stream)
            step(st, st["ws"][1])
        lib.nxv_set_stream(1)
    for i, st in enumerate(sets):
        dl, x, w, labels, _ = xgrad_inputs(torch, name, *shape, seed=10 + i)
        labels[33], x[33], dl[33] = -1, float("nan"), float("nan")
        for t, u in zip(st["in"], (dl, x, w, labels.int())):
            t.copy_(u)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert lib.nxv_synchronize() == 0
    for st in sets:
        got = {k: st[k].clone() for k in ("loss", "dx", "dw")}
        for k in got:
            st[k].fill_(5.0)
        step(st, (None, None))
        torch.cuda.synchronize()
        for k in got:
            assert torch.equal(st[k], got[k]), k
        assert bool(torch.isfinite(got["dw"]).all()) and float(got["loss"][33]) == 0.0
        for room, need in zip(st["ws"][0], st["ws"][2]):
            assert bool((room[need:] == 77).all())
    del graphs


@pytest.mark.parametrize("name", TYPES)
def test_two_threads_on_their_own_streams(nxv, torch, shape, name):
    """Both without a workspace: the library's scratch belongs to the stream."""
    from nx_vulkan_b200 import _native
    lib = _native.load()
    cases = [xgrad_inputs(torch, name, *shape, seed=20 + i) for i in range(2)]
    want = [(xent_run(nxv, torch, *c[1:4], name), xgrad_run(nxv, torch, *c, name)) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            s = torch.cuda.Stream()
            lib.nxv_set_stream(s.cuda_stream)
            with torch.cuda.stream(s):
                for _ in range(20):
                    got = xent_run(nxv, torch, *cases[i][1:4], name), xgrad_run(nxv, torch, *cases[i], name)
                    s.synchronize()
                    if not all(torch.equal(p, q) for a, b in zip(got, want[i]) for p, q in zip(a, b)):
                        wrong.append(i)
                if lib.nxv_synchronize() != 0:
                    wrong.append(_native.last_error())
        except BaseException as e:  # noqa: BLE001
            wrong.append(e)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not wrong, wrong[0]
