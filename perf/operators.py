"""Cases of the operators at the end of a network over classes or tokens: layer norm, dropout and the
softmax cross entropy of a linear layer, each with its gradient.

Where `own` is false, run() computes an operator in its plain form with elementary torch operations in
32 bits (64 for f64 inputs), rounded once at the end.  Where it is true, run() calls nx_vulkan_b200.vulkan on
handles over the same torch tensors (wrap_tensor) and returns the output tensors that the call wrote.

Semantics:
  layer_norm    mean and rstd = 1 / sqrt(var + eps) of every row, y = (x - mean) * rstd * gamma + beta
  dropout       element i is kept, times 1 / (1 - p), when word (offset + i) & 1 of Philox-2x32-10 at counter
                ((offset + i) >> 1, 0) and key seed, shifted right by 8 and taken as a multiple of 2^-24,
                is at least p; the gradient is the same function of the incoming gradient
  cross entropy logits z = x w^T (w: one row per class); lse = log sum_v exp z_v; loss = lse - z_label.
                A label outside [0, vocab) marks a row without a target: loss 0, no gradient.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f64": 8, "bf16": 2}


def listed():
    return [
        # A handful of rows of a small model on its way to an answer: latency.
        {"name": "norm_few_rows_f32", "op": "norm", "dtype": "f32", "rows": 4, "cols": 1000},
        # A ragged batch of an odd width: rows that start at every alignment.
        {"name": "norm_odd_bf16", "op": "norm", "dtype": "bf16", "rows": 2047, "cols": 5001},
        # The tokens of one training step: bandwidth.
        {"name": "norm_step_bf16", "op": "norm", "dtype": "bf16", "rows": 32768, "cols": 4096},
        # The backward pass of a small batch.
        {"name": "norm_grad_small_f32", "op": "norm_grad", "dtype": "f32", "rows": 64, "cols": 1000},
        # A double-precision model: the [4096, 4096] matrix of the reductions' benchmark.
        {"name": "norm_grad_f64", "op": "norm_grad", "dtype": "f64", "rows": 4096, "cols": 4096},
        # The backward pass of one training step.
        {"name": "norm_grad_step_bf16", "op": "norm_grad", "dtype": "bf16", "rows": 16384, "cols": 8192},
        # The activations of a small batch, continuing a stream of random numbers at an odd place.
        {"name": "dropout_small_f32", "op": "dropout", "dtype": "f32", "n": 10007, "p": 0.1, "offset": 4001},
        # The activations of one training step, with an odd tail.
        {"name": "dropout_step_bf16", "op": "dropout", "dtype": "bf16", "n": 134217731, "p": 0.1, "offset": 0},
        # The score of a small batch over a thousand classes.
        {"name": "loss_small_f32", "op": "loss", "dtype": "f32", "n": 64, "vocab": 1001, "dim": 1000},
        # The loss of one training step over a large vocabulary.
        {"name": "loss_step_bf16", "op": "loss", "dtype": "bf16", "n": 8192, "vocab": 65536, "dim": 2048},
        # The gradients of a classifier in single precision with an odd number of classes.
        {"name": "loss_grad_odd_f32", "op": "loss_grad", "dtype": "f32", "n": 2048, "vocab": 10007, "dim": 1000},
        # The gradients of one training step over a large vocabulary.
        {"name": "loss_grad_step_bf16", "op": "loss_grad", "dtype": "bf16", "n": 8192, "vocab": 65536, "dim": 2048},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "dropout", "loss", "loss_grad"])
    if op in ("norm", "norm_grad"):
        cols = _spread(rng, 16, 16384)
        rows = _spread(rng, 1, min(32768, 134217728 // cols))
        dtype = rng.choice(["f32", "f64", "bf16"])
        rows = max(1, rows * 2 // SIZE[dtype])
        return {"op": op, "dtype": dtype, "rows": rows, "cols": cols}
    if op == "dropout":
        dtype = rng.choice(["f32", "f64", "bf16"])
        return {"op": op, "dtype": dtype, "n": _spread(rng, 1, 134217728 * 2 // SIZE[dtype]),
                "p": rng.choice([0.05, 0.1, 0.25, 0.5]), "offset": rng.choice([0, rng.randrange(1 << 24)])}
    return {"op": op, "dtype": rng.choice(["f32", "bf16"]), "n": _spread(rng, 1, 8192),
            "vocab": _spread(rng, 10, 65536), "dim": _spread(rng, 16, 2048)}


def work(case):
    """Each input read once, each output written once, and the products of the formulas."""
    s = SIZE[case["dtype"]]
    if case["op"] == "dropout":
        return {"bytes": 2 * case["n"] * s, "flops": case["n"]}
    if case["op"] in ("norm", "norm_grad"):
        r, c = case["rows"], case["cols"]
        stat = 8 if case["dtype"] == "f64" else 4
        if case["op"] == "norm":
            return {"bytes": 2 * r * c * s + 2 * c * s + 2 * r * stat, "flops": 8 * r * c}
        return {"bytes": 3 * r * c * s + 3 * c * s + 2 * r * stat, "flops": 14 * r * c}
    n, v, d = case["n"], case["vocab"], case["dim"]
    if case["op"] == "loss":
        return {"bytes": (n * d + v * d) * s + 8 * n + 8 * n, "flops": 2 * n * v * d}
    return {"bytes": 2 * (n * d + v * d) * s + 8 * n + 8 * n, "flops": 6 * n * v * d}


def _inputs(case, seed):
    """The call's inputs, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    dt = DTYPES[case["dtype"]]
    wide = torch.float64 if case["dtype"] == "f64" else torch.float32

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale + shift

    if case["op"] == "dropout":
        # activations, a new seed of the mask for every step
        return {"x": normal(case["n"]).to(dt), "seed": (seed * 2654435761 + 12345) % (1 << 32)}
    if case["op"] in ("norm", "norm_grad"):
        r, c = case["rows"], case["cols"]
        # a residual stream: rows of different size, a mean of their own and a few large channels
        channel = 1.0 + 4.0 * (torch.rand(c, generator=g, device="cuda") < 0.01)
        size = torch.exp(normal(r, 1, scale=0.5))
        x = (normal(r, c) * channel * size + normal(r, 1, scale=0.5, shift=0.25)).to(dt)
        s = {"x": x, "gamma": normal(c, scale=0.1, shift=1.0).to(dt), "beta": normal(c, scale=0.1).to(dt)}
        if case["op"] == "norm_grad":
            # what the forward pass left: the statistics of every row
            xw = x.to(wide)
            mean = xw.mean(1)
            s["mean"] = mean
            s["rstd"] = torch.rsqrt((xw - mean[:, None]).square().mean(1) + EPS)
            s["dy"] = normal(r, c, scale=0.01).to(dt)
        return s
    n, v, d = case["n"], case["vocab"], case["dim"]
    # normalised activations; weights that give logits of a standard deviation of about 2
    s = {"x": normal(n, d).to(dt), "w": normal(v, d, scale=2.0 / math.sqrt(d)).to(dt)}
    # few frequent classes and many rare ones; about one row in twenty has no target
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    labels = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp(0, v - 1)
    s["labels"] = torch.where(torch.rand(n, generator=g, device="cuda") < 0.05, -1, labels)
    if case["op"] == "loss_grad":
        # the forward pass's log sum, and the mean over the rows that have a target
        z = s["x"].float() @ s["w"].float().t()
        top = z.amax(1)
        s["lse"] = top + (z - top[:, None]).exp_().sum(1).log()
        del z
        s["dloss"] = torch.full((n,), 1.0, device="cuda") / (s["labels"] >= 0).sum().clamp(min=1)
    return s


def prepare(case, seed):
    state = {"case": case} | _inputs(case, seed)
    if own:
        from nx_vulkan_b200 import _native, vulkan

        if vulkan.init() != "ok":
            raise RuntimeError("no device")
        dt = DTYPES[case["dtype"]]
        wide = torch.float64 if case["dtype"] == "f64" else torch.float32
        new = lambda *shape, dtype=dt: torch.empty(shape, device="cuda", dtype=dtype)  # noqa: E731
        if case["op"] == "dropout":
            outs = [new(case["n"])]
        elif case["op"] == "norm":
            outs = [new(case["rows"], case["cols"]), new(case["rows"], dtype=wide), new(case["rows"], dtype=wide)]
        elif case["op"] == "norm_grad":
            outs = [new(case["rows"], case["cols"]), new(case["cols"]), new(case["cols"])]
        elif case["op"] == "loss":
            outs = [new(case["n"], dtype=torch.float32), new(case["n"], dtype=torch.float32)]
        else:
            outs = [new(case["n"], case["dim"]), new(case["vocab"], case["dim"])]
        # handles over the tensors, as a program that calls the library keeps them
        state["nxv"], state["lib"] = vulkan, _native.load()
        state["outs"] = outs
        state["out"] = tuple(vulkan.wrap_tensor(t) for t in outs)
        state["h"] = {k: vulkan.wrap_tensor(t) for k, t in state.items() if isinstance(t, torch.Tensor)}
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    c, h, out, nxv = state["case"], state["h"], state["out"], state["nxv"]
    state["lib"].nxv_set_stream(torch.cuda.current_stream().cuda_stream or 1)  # 1: the legacy default stream
    if c["op"] == "dropout":
        r = nxv.dropout(h["x"], c["p"], state["seed"], offset=c["offset"], dtype=c["dtype"], out=out[0])
    elif c["op"] == "norm":
        r = nxv.layer_norm(h["x"], h["gamma"], h["beta"], c["rows"], c["cols"], EPS, dtype=c["dtype"], out=out)
    elif c["op"] == "norm_grad":
        r = nxv.layer_norm_grad(h["dy"], h["x"], h["gamma"], h["mean"], h["rstd"], c["rows"], c["cols"],
                                dtype=c["dtype"], out=out)
    elif c["op"] == "loss":
        r = nxv.linear_cross_entropy(h["x"], h["w"], h["labels"], c["n"], c["vocab"], c["dim"],
                                     dtype=c["dtype"], out=out)
    else:
        r = nxv.linear_cross_entropy_grad(h["dloss"], h["x"], h["w"], h["labels"], h["lse"], c["n"], c["vocab"],
                                          c["dim"], dtype=c["dtype"], out=out)
    if r[0] != "ok":
        raise RuntimeError(r[1])
    return state["outs"]


def _round(a, b, key):
    """One round of Philox-2x32 on int64 tensors that hold 32-bit words."""
    mult = 0xD256D193
    high = (a * (mult >> 16) + ((a * (mult & 0xFFFF)) >> 16)) >> 16
    return high ^ key ^ b, (a * mult) & 0xFFFFFFFF


def _words(first, n, seed):
    """Words first .. first + n - 1 of the stream of key seed."""
    key = [(seed + r * 0x9E3779B9) & 0xFFFFFFFF for r in range(10)]
    a = torch.arange(first // 2, (first + n + 1) // 2, device="cuda", dtype=torch.int64)
    b = torch.zeros_like(a)
    a, b = _round(*_round(*_round(*_round(*_round(a, b, key[0]), key[1]), key[2]), key[3]), key[4])
    a, b = _round(*_round(*_round(*_round(*_round(a, b, key[5]), key[6]), key[7]), key[8]), key[9])
    return torch.stack((a, b), 1).reshape(-1)[first % 2:first % 2 + n]


def _run_plain(state):
    c = state["case"]
    dt = DTYPES[c["dtype"]]
    wide = torch.float64 if c["dtype"] == "f64" else torch.float32
    if c["op"] == "dropout":
        x = state["x"].to(wide)
        u = (_words(c["offset"], c["n"], state["seed"]) >> 8).double() * 2.0 ** -24
        return [torch.where(u >= c["p"], x * (1.0 / (1.0 - c["p"])), 0.0).to(dt)]
    if c["op"] == "norm":
        x = state["x"].to(wide)
        mean = x.mean(1)
        centred = x - mean[:, None]
        rstd = 1.0 / (centred.square().mean(1) + EPS).sqrt()
        y = centred * rstd[:, None] * state["gamma"].to(wide) + state["beta"].to(wide)
        return [y.to(dt), mean, rstd]
    if c["op"] == "norm_grad":
        dy, rstd = state["dy"].to(wide), state["rstd"][:, None]
        xhat = (state["x"].to(wide) - state["mean"][:, None]) * rstd
        g = dy * state["gamma"].to(wide)
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        return [dx.to(dt), (dy * xhat).sum(0).to(dt), dy.sum(0).to(dt)]
    x, w, labels = state["x"].float(), state["w"].float(), state["labels"]
    has = (labels >= 0) & (labels < c["vocab"])
    at = labels.clamp(0, c["vocab"] - 1)[:, None]
    z = x @ w.t()
    if c["op"] == "loss":
        top = z.amax(1)
        lse = top + (z - top[:, None]).exp().sum(1).log()
        return [torch.where(has, lse - z.gather(1, at)[:, 0], 0.0), lse]
    p = (z - state["lse"][:, None]).exp()
    p.scatter_(1, at, p.gather(1, at) - 1.0)
    g = torch.where(has[:, None], p * state["dloss"][:, None], 0.0)
    return [(g @ w).to(dt), (g.t() @ torch.where(has[:, None], x, 0.0)).to(dt)]


def exact(case, seed):
    """The outputs in 64 bits, from the definitions."""
    s = _inputs(case, seed)
    d = {k: t.double() for k, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}
    if case["op"] == "dropout":
        n, first = case["n"], case["offset"]
        # Philox on the host, in numpy's unsigned 64-bit numbers, for the sizes where that is quick
        if n > 1 << 24:
            return None
        import numpy as np

        ctr = np.arange(first >> 1, ((first + n - 1) >> 1) + 1, dtype=np.uint64)
        other, key = np.zeros_like(ctr), s["seed"]
        for _ in range(10):
            product = ctr * np.uint64(0xD256D193)
            ctr = (product >> np.uint64(32)) ^ np.uint64(key) ^ other
            other = product & np.uint64(0xFFFFFFFF)
            key = (key + 0x9E3779B9) % (1 << 32)
        words = np.empty(2 * len(ctr), dtype=np.uint64)
        words[0::2], words[1::2] = ctr, other
        words = words[first & 1:][:n] >> np.uint64(8)
        keep = torch.from_numpy(words.astype(np.float64) / 2.0 ** 24 >= case["p"]).cuda()
        return [torch.where(keep, d["x"] / (1.0 - case["p"]), torch.zeros_like(d["x"]))]
    if case["op"] == "norm":
        var, mean = torch.var_mean(d["x"], 1, correction=0)
        rstd = (var + EPS).pow(-0.5)
        y = torch.addcmul(d["beta"], (d["x"] - mean[:, None]) * rstd[:, None], d["gamma"])
        return [y, mean, rstd]
    if case["op"] == "norm_grad":
        n = case["cols"]
        xhat = d["rstd"][:, None] * (d["x"] - d["mean"][:, None])
        g = d["gamma"] * d["dy"]
        along = torch.einsum("rc,rc->r", g, xhat)
        dx = d["rstd"][:, None] / n * (n * g - g.sum(1)[:, None] - along[:, None] * xhat)
        return [dx, torch.einsum("rc,rc->c", d["dy"], xhat), d["dy"].sum(0)]
    labels = s["labels"]
    rows = torch.nonzero((labels >= 0) & (labels < case["vocab"]))[:, 0]
    z = torch.einsum("nd,vd->nv", d["x"], d["w"])
    if case["op"] == "loss":
        lse = torch.logsumexp(z, 1)
        loss = torch.zeros_like(lse)
        loss[rows] = lse[rows] - z[rows, labels[rows]]
        return [loss, lse]
    g = torch.zeros_like(z)
    g[rows] = torch.exp(z[rows] - d["lse"][rows, None])
    g[rows, labels[rows]] -= 1.0
    g *= d["dloss"][:, None]
    x = torch.zeros_like(d["x"])
    x[rows] = d["x"][rows]
    return [torch.einsum("nv,vd->nd", g, d["w"]), torch.einsum("nv,nd->vd", g, x)]
