"""Softmax cross entropy over a vocabulary (laya_vocab_ce_fwd / _bwd) against its definition in 64 bits.

Bounds are the arithmetic's, worst case. A two-piece product holds each operand to 2^-22 and drops a term below 2^-22 of
the product, and adds K terms in fp32, so a sum of products is within (3·2^-22 + K·2^-24)·Σ|a||b| of the exact one. A
logit's error δ moves its probability by p·(δ + δ_lse) and the log-sum-exp by at most the largest δ; exp2 of a rounded
argument and the tiles' sums add a few 2^-23, the stores 2^-24 of the result."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
NO_LABEL = -100
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    from laya_amd.device import Context
    c = Context(0)
    yield c
    c.close()


def _bf16(a):
    """a rounded to bf16 (nearest even): its values and their bit patterns."""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return (r.astype(np.uint32) << 16).view(np.float32), r


def _problem(rows, hidden, vocab, bias=True, labelled=1.0, weighted=False, bf16=False, seed=0, x_scale=1.0):
    r = np.random.default_rng([seed, rows, hidden, vocab])
    W = (r.standard_normal((vocab, hidden)) / np.sqrt(hidden)).astype(np.float32)
    bits = None
    if bf16:
        W, bits = _bf16(W)
    x = (2 * x_scale * r.standard_normal((rows, hidden))).astype(np.float32)
    t = r.integers(0, vocab, rows).astype(np.int32)
    t[r.random(rows) >= labelled] = NO_LABEL
    b = (0.3 * r.standard_normal(vocab)).astype(np.float32) if bias else None
    w = (0.2 + r.random(rows)).astype(np.float32) if weighted else None
    return {"x": x, "W": W, "bits": bits, "t": t, "b": b, "w": w, "scale": 0.37}


def _exact(p):
    """The definition in float64, with the bounds of the module's docstring."""
    x, W = p["x"].astype(np.float64), p["W"].astype(np.float64)
    t, rows, (vocab, hidden) = p["t"], len(p["t"]), p["W"].shape
    has = (t >= 0) & (t < vocab)
    x = np.where(has[:, None], x, 0.0)  # rows without a label are not read
    w = np.where(has, p["w"].astype(np.float64) if p["w"] is not None else 1.0, 0.0)
    z = x @ W.T + (0.0 if p["b"] is None else p["b"].astype(np.float64))
    top = z.max(1, keepdims=True)
    lse = (top + np.log(np.exp(z - top).sum(1, keepdims=True)))[:, 0]
    at = np.where(has, t, 0)
    n = np.arange(rows)
    row_loss = np.where(has, lse - z[n, at], 0.0)
    G = np.exp(z - lse[:, None])
    G[n, at] -= 1.0
    G *= w[:, None] * p["scale"]
    out = {"row_loss": row_loss, "lse": np.where(has, lse, 0.0), "loss": p["scale"] * (w * row_loss).sum(),
           "dx": G @ W, "dW": G.T @ x, "db": G.sum(0)}
    product = lambda a, b, k: (12 * U + k * U) * (np.abs(a) @ np.abs(b))  # noqa: E731
    finite_z = np.where(np.isfinite(z), z, 0.0)
    dz = product(x, W.T, hidden) + 2 * U * np.abs(finite_z)
    dlse = dz.max(1) + 8 * U * (1 + np.abs(lse))
    p_abs = np.exp(z - lse[:, None])
    dG = p_abs * (dz + dlse[:, None] + 4 * U * (2 + np.abs(finite_z - lse[:, None]))) + 4 * U * np.abs(G / np.maximum(
        w * p["scale"], 1e-300)[:, None]) + 2.0 ** -38
    dG *= w[:, None] * p["scale"]
    # row_loss = lse − z_y of the logit that the sum holds: |δ_lse| + |δ_z_y| at most, and the two roundings.
    tol = {"row_loss": dlse + dz[n, at] + 4 * U * (np.abs(lse) + np.abs(np.where(np.isfinite(z[n, at]), z[n, at], 0))),
           "lse": dlse, "dx": dG @ np.abs(W) + product(G, W, vocab) + 4 * U * np.abs(out["dx"]),
           "dW": dG.T @ np.abs(x) + product(G.T, x, rows) + 4 * U * np.abs(out["dW"]),
           "db": dG.sum(0) + (2 + rows) * U * np.abs(G).sum(0) + 4 * U * np.abs(out["db"])}
    tol["loss"] = p["scale"] * (w * tol["row_loss"]).sum() + 4 * U * abs(out["loss"])
    return out, tol


def _run(ctx, p, backward=True, start=None, dx=True):
    """Both calls on the device; `start`: values that dW and db hold before (they accumulate)."""
    from laya_amd import ops
    from laya_amd.device import DeviceArray
    rows, (vocab, hidden) = len(p["t"]), p["W"].shape
    put = lambda a: None if a is None else DeviceArray.from_numpy(ctx, a)  # noqa: E731
    x, t, w = put(p["x"]), put(p["t"]), put(p["w"])
    W = ops.Parameter(ctx, "W", p["W"])
    b = None if p["b"] is None else ops.Parameter(ctx, "b", p["b"])
    w16 = None
    if p["bits"] is not None:
        w16 = DeviceArray(ctx, p["bits"].shape, np.uint16, zero=False)
        w16.upload(p["bits"])
        W.data.fill(float("nan"))  # not read
    guard = 5  # rows behind the last: left as they are
    row_loss, lse = DeviceArray(ctx, (rows + guard,)), DeviceArray(ctx, (rows + guard,))
    loss, bad = DeviceArray(ctx, (1,)), put(np.array([77], np.int32))
    for a in (row_loss, lse):
        a.fill(-3.0)
    ops.vocab_ce(W, b, x, t, rows, row_loss, lse, row_weights=w, scale=p["scale"], loss=loss, weight16=w16,
                 bad_count=bad)
    got = {"row_loss": row_loss.numpy(), "lse": lse.numpy(), "loss": loss.numpy()[0], "bad": bad.numpy()[0]}
    for k in ("row_loss", "lse"):
        assert (got[k][rows:] == -3.0).all(), f"{k} behind the last row was written"
        got[k] = got[k][:rows]
    if backward:
        d = DeviceArray(ctx, (rows + guard, hidden))
        d.fill(7.0)
        if start is not None:
            W.gradient_buffer().upload(start["dW"])
            if b is not None:
                b.gradient_buffer().upload(start["db"])
        ops.vocab_ce_backward(W, b, x, t, rows, lse, d if dx else None, row_weights=w, scale=p["scale"], weight16=w16)
        full = d.numpy()
        assert (full[rows:] == 7.0).all(), "dx behind the last row was written"
        got["dx"], got["dW"] = full[:rows], W.gradient_buffer().numpy()
        if b is not None:
            got["db"] = b.gradient_buffer().numpy()
    return got


def _check(got, want, tol, names=("row_loss", "lse", "loss", "dx", "dW", "db")):
    for k in names:
        if k not in got:
            continue
        off = np.abs(np.asarray(got[k], np.float64) - want[k])
        over = off > tol[k]
        assert not np.any(over | ~np.isfinite(off)), (k, float(np.max(off)), float(np.max(off / np.maximum(tol[k], 1e-300))))


# Rows either side of a block of 16, of the few-row kernels' counts, of their last (256) and of whole tiles; widths and vocabularies that end inside a fragment, a step and a tile.
SHAPES = [(1, 64, 300), (1, 1, 1), (2, 7, 2), (15, 32, 31), (16, 33, 32), (17, 96, 257), (33, 40, 500), (64, 72, 1000),
          (77, 136, 1300), (96, 48, 333), (127, 30, 70), (128, 64, 400), (129, 30, 70), (129, 64, 800), (160, 64, 520),
          (192, 40, 300), (193, 64, 300), (256, 24, 290), (257, 64, 300), (300, 100, 777), (513, 33, 1025), (700, 264, 600)]


@pytest.mark.parametrize("rows,hidden,vocab", SHAPES)
@pytest.mark.parametrize("bf16", [False, True])
def test_matches_the_definition(ctx, rows, hidden, vocab, bf16):
    print(rows, hidden, vocab, bf16, flush=True)
    p = _problem(rows, hidden, vocab, bias=rows % 2 == 0, weighted=rows % 3 == 0, bf16=bf16)
    want, tol = _exact(p)
    got = _run(ctx, p)
    assert got["bad"] == 0
    _check(got, want, tol)


@pytest.mark.parametrize("hidden", [7, 8, 9, 11, 31, 37, 66, 71, 129])
@pytest.mark.parametrize("rows", [13, 90, 210])
def test_widths_that_end_inside_a_load(ctx, rows, hidden):
    """A row of eight, four and two at a time: its last loads start where a whole one still fits."""
    for bf16 in (False, True):
        p = _problem(rows, hidden, 350, weighted=True, bf16=bf16)
        want, tol = _exact(p)
        _check(_run(ctx, p), want, tol)


@pytest.mark.parametrize("rows,hidden,vocab", [(1500, 40, 90), (2100, 264, 300), (5000, 33, 260)])
@pytest.mark.parametrize("labelled", [1.0, 0.1])
def test_many_rows_over_a_small_table(ctx, rows, hidden, vocab, labelled):
    """Few tiles of dW, whose sum over the rows is split, or not, as the labelled rows make it; dW adds to what is there."""
    p = _problem(rows, hidden, vocab, labelled=labelled, weighted=True)
    start = {"dW": np.random.default_rng(2).standard_normal((vocab, hidden)).astype(np.float32),
             "db": np.zeros(vocab, np.float32)}
    want, tol = _exact(p)
    want["dW"] = want["dW"] + start["dW"]
    tol["dW"] = tol["dW"] + 2 * U * np.abs(want["dW"])
    got = _run(ctx, p, start=start)
    _check(got, want, tol)
    again = _run(ctx, p, start=start)
    for k in ("dx", "dW", "db"):
        np.testing.assert_array_equal(got[k], again[k])


@pytest.mark.parametrize("rows,labelled", [(40, 0.5), (250, 0.1), (300, 0.6), (900, 0.15), (600, 0.003), (20, 0.0), (400, 0.0)])
def test_rows_without_a_label_are_not_read(ctx, rows, labelled):
    """NaN and infinite hidden states, weights and all, where no label is: nothing of them reaches a result."""
    p = _problem(rows, 64, 500, labelled=labelled, weighted=True)
    off = p["t"] == NO_LABEL
    p["x"][off] = np.where(np.arange(64) % 2, np.nan, np.inf)
    p["w"][off] = np.nan
    want, tol = _exact({**p, "x": np.where(off[:, None], 0, p["x"]), "w": np.where(off, 0, p["w"])})
    got = _run(ctx, p)
    _check(got, want, tol)
    assert (got["row_loss"][off] == 0).all() and (got["lse"][off] == 0).all() and (got["dx"][off] == 0).all()


def test_targets_outside_the_vocabulary_are_counted_and_ignored(ctx):
    for rows in (50, 400):
        p = _problem(rows, 64, 300, labelled=0.8)
        p["t"][3], p["t"][7], p["t"][9] = 300, -1, 2 ** 30
        got = _run(ctx, p)
        assert got["bad"] == 3
        want, tol = _exact(p)
        _check(got, want, tol)


@pytest.mark.parametrize("rows", [30, 330])
def test_gradients_accumulate_and_dx_is_overwritten(ctx, rows):
    p = _problem(rows, 64, 300)
    r = np.random.default_rng(1)
    start = {"dW": r.standard_normal((300, 64)).astype(np.float32), "db": r.standard_normal(300).astype(np.float32)}
    want, tol = _exact(p)
    got = _run(ctx, p, start=start)
    for k in ("dW", "db"):
        want[k] = want[k] + start[k]
        tol[k] = tol[k] + 2 * U * np.abs(want[k])
    _check(got, want, tol)


@pytest.mark.parametrize("rows", [30, 330])
def test_entries_masked_by_the_bias(ctx, rows):
    """b = −∞ leaves an entry out (its probability and gradient are 0), the type's lowest value as good as that."""
    p = _problem(rows, 64, 700)
    mask = np.arange(700) % 3 == 1
    p["b"][mask] = -np.inf
    p["b"][600:] = np.finfo(np.float32).min
    mask[600:] = True
    allowed = np.flatnonzero(~mask)
    p["t"] = allowed[p["t"] % len(allowed)].astype(np.int32)
    exact = {**p, "b": np.where(mask, -np.inf, p["b"])}
    with np.errstate(invalid="ignore"):
        want, tol = _exact(exact)
    got = _run(ctx, p)
    _check(got, want, tol)
    assert (got["dW"][mask] == 0).all() and (got["db"][mask] == 0).all()


@pytest.mark.parametrize("rows", [30, 330])
def test_a_row_with_nothing_allowed_is_nan_and_no_other_is(ctx, rows):
    """Every entry masked: log-sum-exp −∞, the loss (−∞) − (−∞). A non-finite hidden state: its own row alone."""
    p = _problem(rows, 64, 300)
    p["x"][5, 3] = np.inf
    p["x"][8] = np.nan
    got = _run(ctx, p, backward=False)
    others = np.ones(rows, bool)
    others[[5, 8]] = False
    want, tol = _exact({**p, "x": np.where(others[:, None], p["x"], 0)})
    assert not np.isfinite(got["row_loss"][~others]).any() and np.isnan(got["loss"])
    for k in ("row_loss", "lse"):
        assert (np.abs(got[k] - want[k]) <= tol[k])[others].all()
    p = _problem(rows, 64, 300)
    p["b"][:] = -np.inf
    got = _run(ctx, p, backward=False)
    assert np.isnan(got["row_loss"]).all() and np.isneginf(got["lse"]).all()


@pytest.mark.parametrize("rows", [40, 340])
def test_magnitudes_far_apart(ctx, rows):
    """Rows of x from 1e-30 to 1e4 (each has its scale) and a table whose columns grow by 2^40 along a row (the few-row
    kernels' running scale moves many times), with logits still of order one: the bounds hold row by row."""
    p = _problem(rows, 96, 400)
    grow = 2.0 ** np.linspace(-30, 10, 96)
    p["W"] = (p["W"] * grow).astype(np.float32)
    p["x"] = (p["x"] / grow).astype(np.float32)
    p["x"][:10] *= np.float32(1e-25)
    # A two-piece operand holds values below 2^-18 of its scale's largest to 2^-40 of that: a product with the other
    # side's largest, K of them.
    want, tol = _exact(p)
    floor = 2.0 ** -36 * 96 * np.abs(p["x"]).max(1) * np.abs(p["W"]).max()
    for k in ("row_loss", "lse"):
        tol[k] = tol[k] + 2 * floor
    got = _run(ctx, p, backward=False)
    _check(got, want, tol, ("row_loss", "lse"))


def test_zero_weight_and_hidden_rows(ctx):
    for rows in (20, 300):
        p = _problem(rows, 64, 300)
        p["W"][10:200] = 0
        p["x"][3] = 0
        want, tol = _exact(p)
        _check(_run(ctx, p), want, tol)
        p["W"][:] = 0
        want, tol = _exact(p)
        _check(_run(ctx, p), want, tol)


@pytest.mark.parametrize("rows", [30, 150, 250, 330, 1400])
@pytest.mark.parametrize("bf16", [False, True])
def test_small_losses_of_large_logits(ctx, rows, bf16):
    """A target ahead of the next entry by ten, with logits of 200: loss = log(1 + s), s = Σ_{v ≠ y} exp(z_v − z_y). The
    target's logit is in the sum as it is subtracted, so its own error e moves the loss by e·s / (1 + s), as the others'
    do: 2·e·s in all. Beside that the sum is near one and is off by a few roundings: of up to 32 values a lane, 6 exchanges
    and as many merges, 64·U."""
    p = _problem(rows, 256, 600, bias=False)
    p["W"][1::2] = np.float32(0.95) * p["W"][::2]
    if bf16:
        p["W"], p["bits"] = _bf16(p["W"])
    p["t"] = (p["t"] // 2 * 2).astype(np.int32)
    target = p["W"][p["t"]].astype(np.float64)
    p["x"] = (200 * target / (target ** 2).sum(1, keepdims=True)).astype(np.float32)
    W, x = p["W"].astype(np.float64), p["x"].astype(np.float64)
    z, off = x @ W.T, (12 * U + 256 * U) * (np.abs(x) @ np.abs(W).T)
    n = np.arange(rows)
    d = z - z[n, p["t"]][:, None]
    d[n, p["t"]] = -np.inf
    s = np.exp(d).sum(1)
    got = _run(ctx, p, backward=False)
    assert (np.abs(got["row_loss"] - np.log1p(s)) <= 2 * s * (off + 2 * U * np.abs(z)).max(1) + 64 * U).all()


@pytest.mark.parametrize("rows", [77, 600])
def test_two_runs_give_the_same_bits_and_so_does_a_warm_workspace(ctx, rows):
    p = _problem(rows, 104, 900, weighted=True, labelled=0.9)
    a = _run(ctx, p)
    _run(ctx, _problem(1200, 64, 300))  # leaves other values in the workspace
    b = _run(ctx, p)
    for k in ("row_loss", "lse", "loss", "dx", "dW", "db"):
        np.testing.assert_array_equal(a[k], b[k])


def test_rows_that_need_no_gradient_of_x(ctx):
    for rows in (40, 400):
        p = _problem(rows, 64, 300)
        want, tol = _exact(p)
        _check(_run(ctx, p, dx=False), want, tol, ("dW", "db"))


def test_frozen_weight(ctx):
    """A weight that is not trainable gets no gradient; dx stays the same bits."""
    from laya_amd import ops
    from laya_amd.device import DeviceArray
    for rows in (40, 400):
        p = _problem(rows, 64, 300)
        all_of = _run(ctx, p)
        W, b = ops.Parameter(ctx, "W", p["W"], trainable=False), ops.Parameter(ctx, "b", p["b"], trainable=False)
        x, t = DeviceArray.from_numpy(ctx, p["x"]), DeviceArray.from_numpy(ctx, p["t"])
        lse, dx = DeviceArray.from_numpy(ctx, all_of["lse"]), DeviceArray(ctx, (rows, 64))
        ops.vocab_ce_backward(W, b, x, t, rows, lse, dx, scale=p["scale"])
        assert W.gradient is None and b.gradient is None
        off = np.abs(dx.numpy() - all_of["dx"])
        assert off.max() <= 64 * U * np.abs(all_of["dx"]).max()  # dx's sum may be split another way: a few roundings


def test_no_rows(ctx):
    p = _problem(0, 64, 300)
    got = _run(ctx, p)
    assert got["loss"] == 0 and got["bad"] == 0 and (got["dW"] == 0).all()


def test_unaligned_table_and_states(ctx):
    """A table and states that start 4 bytes off a 16-byte boundary (views into an arena)."""
    from laya_amd import ops
    from laya_amd.device import DeviceArray
    for rows in (40, 400):
        p = _problem(rows, 64, 300)
        arena = DeviceArray(ctx, (2 * 300 * 64 + rows * 64 * 2 + 64,))
        at = [1]

        def view(a, shape):
            v = DeviceArray.borrow(ctx, arena.ptr + 4 * at[0], shape, owner=arena)
            at[0] += (int(np.prod(shape)) + 3) // 4 * 4
            if a is not None:
                v.upload(a)
            return v

        W = ops.Parameter.borrow(ctx, "W", (300, 64), view(p["W"], (300, 64)), view(None, (300, 64)))
        b = ops.Parameter(ctx, "b", p["b"])
        x, dx = view(p["x"], (rows, 64)), view(None, (rows, 64))
        t = DeviceArray.from_numpy(ctx, p["t"])
        row_loss, lse = DeviceArray(ctx, (rows,)), DeviceArray(ctx, (rows,))
        ops.vocab_ce(W, b, x, t, rows, row_loss, lse, scale=p["scale"])
        ops.vocab_ce_backward(W, b, x, t, rows, lse, dx, scale=p["scale"])
        want, tol = _exact(p)
        _check({"row_loss": row_loss.numpy(), "lse": lse.numpy(), "dx": dx.numpy(), "dW": W.gradient.numpy(),
                "db": b.gradient.numpy()}, want, tol)


@pytest.mark.parametrize("rows", [5, 300])
def test_a_table_of_more_than_2_31_values(ctx, rows):
    """1,100,000 x 2048: zeros but for the last 64 rows, which lie past an int's range of elements. A row's logits are then
    64 numbers and zeros, whose exponentials, ones, add without error."""
    from laya_amd import ops
    from laya_amd.device import DeviceArray
    vocab, hidden, last = 1_100_000, 2048, 64
    r = np.random.default_rng(rows)
    x = r.standard_normal((rows, hidden)).astype(np.float32)
    w = (r.standard_normal((last, hidden)) * 4 / np.sqrt(hidden)).astype(np.float32)
    t = (vocab - 1 - r.integers(0, last, rows)).astype(np.int32)
    W, dW = DeviceArray(ctx, (vocab, hidden)), DeviceArray(ctx, (vocab, hidden))
    try:
        W.fill(0.0)
        dW.fill(0.0)
        part = lambda a, v: DeviceArray.borrow(ctx, a.ptr + 4 * v * hidden, (last, hidden), owner=a)  # noqa: E731
        part(W, vocab - last).upload(w)
        P = ops.Parameter.borrow(ctx, "W", (vocab, hidden), W, dW)
        X, T, dx = DeviceArray.from_numpy(ctx, x), DeviceArray.from_numpy(ctx, t), DeviceArray(ctx, (rows, hidden))
        row_loss, lse = DeviceArray(ctx, (rows,)), DeviceArray(ctx, (rows,))
        ops.vocab_ce(P, None, X, T, rows, row_loss, lse, scale=0.5)
        ops.vocab_ce_backward(P, None, X, T, rows, lse, dx, scale=0.5)
        xd, wd, n = x.astype(np.float64), w.astype(np.float64), np.arange(rows)
        z, at = xd @ wd.T, t - (vocab - last)
        want = np.log(vocab - last + np.exp(z).sum(1))
        dz = (12 * U + hidden * U) * (np.abs(xd) @ np.abs(wd).T) + 2 * U * np.abs(z)
        off = dz.max(1) + 8 * U * (1 + np.abs(want))
        assert (np.abs(lse.numpy() - want) <= off).all()
        assert (np.abs(row_loss.numpy() - (want - z[n, at])) <= off + dz[n, at] + 8 * U * np.abs(want)).all()
        p = np.exp(z - want[:, None])
        G = 0.5 * p
        G[n, at] -= 0.5
        dG = 0.5 * p * (dz + off[:, None] + 4 * U * (2 + np.abs(z - want[:, None]))) + 4 * U * np.abs(G) + 2.0 ** -38
        sums = lambda a, b, k: (12 + k) * U * (np.abs(a) @ np.abs(b))  # noqa: E731
        assert (np.abs(dx.numpy() - G @ wd) <= dG @ np.abs(wd) + sums(G, wd, 2 * last) + 4 * U * np.abs(G @ wd)).all()
        got = part(dW, vocab - last).numpy()
        assert (np.abs(got - G.T @ xd) <= dG.T @ np.abs(xd) + sums(G.T, xd, rows) + 4 * U * np.abs(G.T @ xd)).all()
        G0 = 0.5 * np.exp(-want)[:, None] * np.ones(last)  # rows of zeros, one side and the other of 2^31 values
        dG0 = G0 * (off[:, None] + 4 * U * (2 + np.abs(want[:, None]))) + 2.0 ** -38
        for v in (0, 2 ** 31 // hidden - last // 2, vocab - 2 * last):
            got = part(dW, v).numpy()
            assert (np.abs(got - G0.T @ xd) <= dG0.T @ np.abs(xd) + sums(G0.T, xd, rows) + 4 * U * np.abs(G0.T @ xd)).all()
    finally:
        W.free()
        dW.free()


@pytest.mark.parametrize("rows", [24, 280])
def test_gradient_against_differences_of_the_loss(ctx, rows):
    """Central differences of the device's own loss along random directions. With step h the quotient is off by
    2·err(loss)/2h and by h²/6 of the third derivative along the direction, which for a log-sum-exp is at most the cube
    of the logits' change per unit of h."""
    p = _problem(rows, 48, 200, weighted=True)
    r = np.random.default_rng(3)
    got = _run(ctx, p)
    _, tol = _exact(p)
    for what, grad in (("x", "dx"), ("W", "dW"), ("b", "db")):
        d = r.standard_normal(p[what].shape)
        h = 2.0 ** -5
        step = {"x": lambda s: p["x"] + s * h * d, "W": lambda s: p["W"] + s * h * d, "b": lambda s: p["b"] + s * h * d}[what]
        loss = [_run(ctx, {**p, what: step(s).astype(np.float32)}, backward=False)["loss"].astype(np.float64)
                for s in (1, -1)]
        moved = {"x": lambda: np.abs(d @ p["W"].T).max(1), "W": lambda: np.abs(p["x"] @ d.T).max(1),
                 "b": lambda: np.full(rows, np.abs(d).max())}[what]()
        third = p["scale"] * (p["w"] * (2 * moved) ** 3).sum()
        rounding = 2.0 ** -24 * np.abs(step(1)).max() / h * np.abs(got[grad]).sum()  # of the moved operand
        allowed = 2 * tol["loss"] / h + h * h / 6 * third + 2 * rounding + 1e-5 * np.abs(got[grad] * d).sum()
        assert abs((loss[0] - loss[1]) / (2 * h) - (got[grad] * d).sum()) <= allowed, what


@pytest.mark.parametrize("rows,vocab", [(300, 5003), (700, 2600)])
def test_a_vocabulary_of_several_pieces(rows, vocab):
    """Under a memory cap the vocabulary goes through in pieces of what the cap leaves (without one, of 3 GiB)."""
    from laya_amd.device import Context
    p = _problem(rows, 100, vocab, weighted=True, labelled=0.9)
    want, tol = _exact(p)
    capped = Context(0)
    try:
        # The arrays of _run (the table and its gradient, x and dx, small ones), then 3 MiB: half of it is far less than
        # the packed table and G (4 · vocab · (104 + rows) bytes or more) take at once.
        capped.set_memory_cap(2 * 4 * vocab * 100 + 2 * 4 * rows * 100 + (4 << 20) + 12 * rows * 100 * 4)
        _check(_run(capped, p), want, tol)
    finally:
        capped.close()


def test_two_contexts_at_once(ctx):
    """Calls on two contexts, each with its stream and workspace, started before either is waited for."""
    from laya_amd.device import Context
    other = Context(0)
    try:
        for rows in (60, 500):
            p, q = _problem(rows, 64, 2000, seed=1), _problem(rows + 9, 64, 2000, seed=2)
            a, b = _run(ctx, p), _run(other, q)
            for got, prob in ((a, p), (b, q)):
                want, tol = _exact(prob)
                _check(got, want, tol)
    finally:
        other.close()


def test_refusals(ctx):
    """Calls that the library refuses before any launch."""
    from laya_amd import ops
    from laya_amd._native import ERR_ARGUMENT, lib
    from laya_amd.device import DeviceArray
    L = lib()
    a = DeviceArray(ctx, (64,))
    f = ctypes.c_float(1.0)
    good = [ctx.handle, a.ptr, 2, 4, a.ptr, None, 8, None, a.ptr, None, f, a.ptr, a.ptr, None, None]
    for at, value in ((1, None), (2, -1), (3, 0), (4, None), (6, 0), (8, None), (11, None), (12, None), (2, 1 << 23),
                      (3, 1 << 17), (6, 1 << 25), (10, ctypes.c_float(float("nan")))):
        args = list(good)
        args[at] = value
        assert L.laya_vocab_ce_fwd(*args) == ERR_ARGUMENT, at
    good = [ctx.handle, a.ptr, 2, 4, a.ptr, None, 8, None, a.ptr, None, f, a.ptr, a.ptr, None, None]
    for at, value in ((1, None), (3, 0), (8, None), (11, None), (12, a.ptr)):
        args = list(good)
        args[at] = value
        assert L.laya_vocab_ce_bwd(*args) == ERR_ARGUMENT, at
    W = ops.Parameter(ctx, "W", np.zeros((8, 4), np.float32))
    with pytest.raises(ValueError):
        ops.vocab_ce(W, None, a, DeviceArray.from_numpy(ctx, np.zeros(64, np.int32)), 20, a, a)
