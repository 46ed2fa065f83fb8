"""Newton-Schulz orthogonalisation and the Muon step (laya_orthogonalize, laya_muon) against the iteration in 64 bits.

The products carry fp32 accuracy (two fp16 pieces), so a result may be as far from the exact iteration as the same
iteration in fp32 is, a few times: each of the three products of a step rounds its operands to 2^-22 where fp32 rounds to
2^-24, on top of sums of the same length. Bound: four times the fp32 iteration's own error, plus 2^-19 (one step's
roundings, 3·2^-22 a product, through a quintic whose slope is at most 4.3)."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
A, B, C = 3.4445, -4.7750, 2.0315


@pytest.fixture(scope="module")
def ctx():
    from laya_amd.device import Context
    c = Context(0)
    yield c
    c.close()


def _iterate(u, steps, dtype):
    """The definition, in dtype; norms in 64 bits."""
    x = np.asarray(u, np.float64)
    n = np.sqrt((x ** 2).sum())
    x = (x / n if n else x).astype(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.T.copy() if tall else x
    a, b, c = (dtype(v) for v in (A, B, C))
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.T if tall else x


def _close(got, u, steps, scale=1.0):
    want = _iterate(u, steps, np.float64) * scale
    own = np.linalg.norm(_iterate(u, steps, np.float32) * scale - want)
    off = np.linalg.norm(got - want)
    assert off <= 4 * own + 2.0 ** -19 * np.linalg.norm(want), (off / max(np.linalg.norm(want), 1e-300), own)


def _matrices(count, rows, cols, seed=0, rank=None):
    r = np.random.default_rng([seed, count, rows, cols])
    u = r.standard_normal((count, rows, cols))
    if rank:
        u = np.einsum("nik,nkj->nij", r.standard_normal((count, rows, rank)), r.standard_normal((count, rank, cols)))
    return (u * np.exp(0.5 * r.standard_normal((1, 1, cols)))).astype(np.float32)


def _orthogonalize(ctx, u, steps=5, in_place=False):
    from laya_amd import ops
    from laya_amd.device import DeviceArray
    x = DeviceArray.from_numpy(ctx, u)
    out = x if in_place else DeviceArray(ctx, (u.size + 3,))
    if not in_place:
        out.fill(9.0)
    ops.orthogonalize(ctx, x, *u.shape, out, steps=steps)
    got = out.numpy().reshape(-1)
    if not in_place:
        assert (got[u.size:] == 9.0).all(), "written behind the last matrix"
        np.testing.assert_array_equal(x.numpy(), u)  # the input is left as it was
    return got[:u.size].reshape(u.shape)


@pytest.mark.parametrize("count,rows,cols", [(1, 1, 1), (2, 1, 5), (2, 5, 1), (3, 17, 17), (2, 32, 64), (1, 33, 70), (4, 70, 33),
                                             (2, 128, 300), (2, 300, 128), (1, 257, 256), (1, 260, 700), (40, 64, 96),
                                             (3, 513, 130), (1, 768, 768)])
def test_matches_the_iteration(ctx, count, rows, cols):
    print(count, rows, cols, flush=True)
    u = _matrices(count, rows, cols)
    got = _orthogonalize(ctx, u)
    for k in range(count):
        _close(got[k], u[k], 5)


@pytest.mark.parametrize("steps", [1, 2, 7])
def test_other_numbers_of_steps(ctx, steps):
    for shape in ((2, 60, 90), (1, 90, 60)):
        u = _matrices(*shape)
        got = _orthogonalize(ctx, u, steps)
        for k in range(shape[0]):
            _close(got[k], u[k], steps)


@pytest.mark.parametrize("count,rows,cols", [(60, 300, 400), (60, 400, 300), (16, 1100, 1056), (10, 1056, 3100)])
def test_many_tiles(ctx, count, rows, cols):
    """Enough matrices for each size of tile (256 wide ones in the last two), ending inside them, in both orders."""
    u = _matrices(count, rows, cols)
    got = _orthogonalize(ctx, u)
    for k in (0, count - 1):
        _close(got[k], u[k], 5)


def test_singular_values_gather_near_one(ctx):
    u = _matrices(1, 200, 320)
    s = np.linalg.svd(_orthogonalize(ctx, u)[0].astype(np.float64), compute_uv=False)
    assert s.min() > 0.3 and s.max() < 1.25  # values above 1/400 of the norm reach [0.68, 1.21] in five steps


def test_low_rank_and_zero_matrices(ctx):
    u = _matrices(3, 96, 200, rank=4)
    u[1] = 0
    got = _orthogonalize(ctx, u)
    assert (got[1] == 0).all()
    _close(got[0], u[0], 5)
    _close(got[2], u[2], 5)


def test_the_norm_of_the_input_does_not_matter(ctx):
    """Powers of two change nothing but the norm, which is divided out in 64 bits; 1e-30 and 1e30 neither under- nor
    overflow in its sum of squares."""
    u = _matrices(1, 64, 100)
    base = _orthogonalize(ctx, u)
    for e in (-100, -20, 20, 100):
        np.testing.assert_array_equal(_orthogonalize(ctx, u * np.float32(2.0 ** e)), base)


def test_a_matrix_that_is_not_finite_spoils_itself_alone(ctx):
    for bad in (np.nan, np.inf):
        u = _matrices(3, 40, 64)
        clean = _orthogonalize(ctx, u)
        u[1, 3, 5] = bad
        got = _orthogonalize(ctx, u)
        assert not np.isfinite(got[1]).any()
        np.testing.assert_array_equal(got[[0, 2]], clean[[0, 2]])


def test_in_place_and_again(ctx):
    for shape in ((2, 60, 90), (3, 90, 60), (1, 300, 300)):
        u = _matrices(*shape)
        a = _orthogonalize(ctx, u)
        _orthogonalize(ctx, _matrices(2, 200, 333))  # leaves other values in the workspace
        np.testing.assert_array_equal(_orthogonalize(ctx, u), a)
        np.testing.assert_array_equal(_orthogonalize(ctx, u, in_place=True), a)


def test_no_matrices(ctx):
    from laya_amd import ops
    from laya_amd.device import DeviceArray
    ops.orthogonalize(ctx, DeviceArray(ctx, (4,)), 0, 5, 5, DeviceArray(ctx, (4,)))


# ------------------------------------------------------------------------------------------ the step

SHAPES = [(48, 16), (16, 16), (40, 64), (16, 48), (48, 16), (33, 7), (1, 9), (64, 40), (16, 48)]


def _arena(shapes, gap, seed=0):
    r = np.random.default_rng(seed)
    offsets, at = [], 3
    for rows, cols in shapes:
        offsets.append(at)
        at += rows * cols + gap
    p, g, m = (r.standard_normal(at + 11).astype(np.float32) * s for s in (0.05, 1e-3, 4e-3))
    return offsets, p, g, m


def _step(ctx, shapes, offsets, p, g, m, multipliers=None, coef=None, times=1, **kw):
    from laya_amd import ops
    from laya_amd.device import DeviceArray
    mats = ops.MuonMatrices(ctx, offsets, [s[0] for s in shapes], [s[1] for s in shapes], multipliers)
    P, G, M = (DeviceArray.from_numpy(ctx, a) for a in (p, g, m))
    c = None if coef is None else DeviceArray.from_numpy(ctx, np.array([coef], np.float32))
    for _ in range(times):
        ops.muon(mats, P, G, M, coef=c, **kw)
    out = P.numpy(), G.numpy(), M.numpy()
    mats.close()
    return out


def _reference(shapes, offsets, p, g, m, multipliers=None, coef=1.0, learning_rate=0.0, mu=0.95, nesterov=True,
               weight_decay=0.0, steps=5, zero_grads=False, dtype=np.float64):
    p, g, m = p.astype(np.float64), g.astype(np.float64), m.astype(np.float64)
    for i, (rows, cols) in enumerate(shapes):
        at = slice(offsets[i], offsets[i] + rows * cols)
        m[at] = mu * m[at] + coef * g[at]
        u = coef * g[at] + mu * m[at] if nesterov else m[at]
        k = 1.0 if multipliers is None else multipliers[i]
        x = _iterate(u.reshape(rows, cols), steps, dtype).astype(np.float64).reshape(-1)
        p[at] = p[at] * (1 - learning_rate * weight_decay) - learning_rate * k * x
        if zero_grads:
            g[at] = 0
    return p, g, m


@pytest.mark.parametrize("gap", [0, 4, 5])
@pytest.mark.parametrize("nesterov", [True, False])
def test_step_matches_the_formula(ctx, gap, nesterov):
    """Matrices of many shapes in one arena, some off 16-byte boundaries; what lies between them is left alone."""
    offsets, p, g, m = _arena(SHAPES, gap)
    mult = [0.5 + 0.25 * i for i in range(len(SHAPES))]
    kw = dict(learning_rate=0.02, mu=0.9, nesterov=nesterov, weight_decay=0.1)
    P, G, M = _step(ctx, SHAPES, offsets, p, g, m, mult, coef=0.75, zero_grads=True, **kw)
    wp, wg, wm = _reference(SHAPES, offsets, p, g, m, mult, coef=0.75, zero_grads=True, **kw)
    own, _, _ = _reference(SHAPES, offsets, p, g, m, mult, coef=0.75, dtype=np.float32, **kw)
    np.testing.assert_allclose(M, wm, rtol=2.0 ** -22, atol=2.0 ** -22 * np.abs(m).max())  # two roundings
    np.testing.assert_array_equal(G, wg.astype(np.float32))
    inside = np.zeros(len(p), bool)
    for i, (rows, cols) in enumerate(SHAPES):
        at = slice(offsets[i], offsets[i] + rows * cols)
        inside[at] = True
        moved = np.linalg.norm(wp[at] - p[at])
        off = np.linalg.norm(P[at] - wp[at])
        assert off <= 4 * np.linalg.norm(own[at] - wp[at]) + 2.0 ** -19 * moved + 2.0 ** -23 * np.linalg.norm(p[at]), i
    for got, before in ((P, p), (G, g), (M, m)):
        np.testing.assert_array_equal(got[~inside], before[~inside])


def test_gradients_are_kept_unless_cleared_and_steps_follow_one_another(ctx):
    offsets, p, g, m = _arena(SHAPES[:3], 0)
    kw = dict(learning_rate=0.02, weight_decay=0.01)
    P, G, M = _step(ctx, SHAPES[:3], offsets, p, g, m, times=2, **kw)
    np.testing.assert_array_equal(G, g)
    once = _step(ctx, SHAPES[:3], offsets, p, g, m, **kw)
    twice = _step(ctx, SHAPES[:3], offsets, once[0], g, once[2], **kw)
    np.testing.assert_array_equal(P, twice[0])
    np.testing.assert_array_equal(M, twice[2])


def test_more_shapes_than_a_launch_names(ctx):
    shapes = [(16 + i, 24) for i in range(21)] + [(24, 16 + i) for i in range(1, 20)]
    offsets, p, g, m = _arena(shapes, 1)
    kw = dict(learning_rate=0.1)
    P, _, _ = _step(ctx, shapes, offsets, p, g, m, **kw)
    wp, _, _ = _reference(shapes, offsets, p, g, m, **kw)
    for i, (rows, cols) in enumerate(shapes):
        at = slice(offsets[i], offsets[i] + rows * cols)
        assert np.linalg.norm(P[at] - wp[at]) <= 2.0 ** -16 * np.linalg.norm(wp[at] - p[at]) + 2.0 ** -23 * np.linalg.norm(p[at])


def test_zero_momentum_and_gradient_only_decays(ctx):
    offsets, p, g, m = _arena(SHAPES, 0)
    P, _, M = _step(ctx, SHAPES, offsets, p, 0 * g, 0 * m, learning_rate=0.5, weight_decay=0.25)
    assert (M == 0).all()
    for i, (rows, cols) in enumerate(SHAPES):
        at = slice(offsets[i], offsets[i] + rows * cols)
        np.testing.assert_array_equal(P[at], p[at] * np.float32(1 - 0.5 * 0.25))


def test_refusals(ctx):
    from laya_amd import ops
    from laya_amd._native import ERR_ARGUMENT, LayaArgumentError, lib
    from laya_amd.device import DeviceArray
    L = lib()
    a, b, c = (DeviceArray(ctx, (64,)) for _ in range(3))
    for args in ((None, 1, 4, 4, 5, b.ptr), (a.ptr, 1, 0, 4, 5, b.ptr), (a.ptr, 1, 4, -1, 5, b.ptr), (a.ptr, -1, 4, 4, 5, b.ptr),
                 (a.ptr, 1, 4, 4, 0, b.ptr), (a.ptr, 1, 4, 4, 101, b.ptr), (a.ptr, 1, 4, 4, 5, None),
                 (a.ptr, 1, 1 << 20, 1 << 20, 5, b.ptr)):
        assert L.laya_orthogonalize(ctx.handle, *args) == ERR_ARGUMENT, args
    with pytest.raises(LayaArgumentError, match="overlap"):
        ops.MuonMatrices(ctx, [0, 10], [4, 2], [4, 2])
    with pytest.raises(LayaArgumentError, match="overlap"):
        ops.MuonMatrices(ctx, [8, 8], [2, 2], [2, 2])
    with pytest.raises(LayaArgumentError):
        ops.MuonMatrices(ctx, [0], [0], [2])
    with pytest.raises(LayaArgumentError, match="finite"):
        ops.MuonMatrices(ctx, [0], [2], [2], [float("inf")])
    m = ops.MuonMatrices(ctx, [0, 16], [4, 4], [4, 4])
    f = [m.handle, a.ptr, b.ptr, c.ptr, ctypes.c_double(0.1), ctypes.c_double(0.9), 1, ctypes.c_double(0.0), 5, None, 0]
    nan = ctypes.c_double(float("nan"))
    for at, value in ((0, None), (1, None), (2, a.ptr), (3, b.ptr), (4, nan), (5, ctypes.c_double(1.0)),
                      (5, ctypes.c_double(-0.1)), (7, nan), (8, 0)):
        args = list(f)
        args[at] = value
        assert L.laya_muon(ctx.handle, *args) == ERR_ARGUMENT, at
    with pytest.raises(ValueError):
        ops.muon(m, a, b, DeviceArray(ctx, (20,)), 0.1)


@pytest.mark.parametrize("rows,cols", [(1048575, 2048), (2048, 1048575), (46341, 46341), (1 << 20, 1 << 20)])
def test_sizes_past_an_int_are_refused(ctx, rows, cols):
    """2^31 elements, and the last few below it, where the ends of the norm's chunks would not fit an int."""
    from laya_amd import ops
    from laya_amd._native import ERR_ARGUMENT, LayaArgumentError, lib
    from laya_amd.device import DeviceArray
    a = DeviceArray(ctx, (64,))
    assert lib().laya_orthogonalize(ctx.handle, a.ptr, 1, rows, cols, 5, a.ptr) == ERR_ARGUMENT
    with pytest.raises(LayaArgumentError, match=f"{rows} x {cols}"):
        ops.MuonMatrices(ctx, [0], [rows], [cols])


def test_matrices_of_another_context(ctx):
    """The tables are on the device when the call returns: another context's stream may read them at once."""
    from laya_amd import ops
    from laya_amd.device import Context, DeviceArray
    r = np.random.default_rng(4)
    p, g = (r.standard_normal(24 * 40).astype(np.float32) for _ in range(2))
    out = []
    other = Context(ctx.device)
    try:
        for run in (ctx, other):
            P, G, M = (DeviceArray.from_numpy(run, v) for v in (p, g, np.zeros_like(p)))
            run.sync()
            m = ops.MuonMatrices(ctx, [0], [24], [40])
            m.ctx = run
            ops.muon(m, P, G, M, 0.1)
            out.append(P.numpy())
            m.ctx = ctx
    finally:
        other.close()
    np.testing.assert_array_equal(out[0], out[1])


def test_no_matrices_to_move(ctx):
    from laya_amd import ops
    from laya_amd.device import DeviceArray
    a, b, c = (DeviceArray(ctx, (4,)) for _ in range(3))
    ops.muon(ops.MuonMatrices(ctx, [], [], []), a, b, c, 0.1)


# ------------------------------------------------------------- a step of masked-token training, all together

def test_a_step_of_masked_token_training(ctx):
    """Embeddings, a linear layer, a LayerNorm, the vocabulary loss on the tied table, and back; then the clip, a Muon step
    of the layer's matrix and an AdamW step of the rest, three times over, beside the same in 64 bits. The two
    trajectories part by fp32 rounding: relative errors of a few 2^-22 a step in gradients and update, 2^-15 allowed."""
    from laya_amd import ops
    from laya_amd._native import check, lib
    from laya_amd.device import DeviceArray
    L = lib()
    r = np.random.default_rng(11)
    V, H, T, lr, eps = 400, 64, 300, 0.02, 1e-5
    sizes = {"E": (V, H), "M": (H, H), "gamma": (H,), "bias": (V,)}
    offsets, at = {}, 0
    for k, s in sizes.items():
        offsets[k] = at
        at += int(np.prod(s))
    p0 = {"E": 0.1 * r.standard_normal((V, H)), "M": np.eye(H) + 0.1 * r.standard_normal((H, H)),
          "gamma": 1 + 0.1 * r.standard_normal(H), "bias": 0.1 * r.standard_normal(V)}
    flat = np.concatenate([p0[k].reshape(-1) for k in sizes]).astype(np.float32)
    P, G, M1, M2 = (DeviceArray.from_numpy(ctx, flat if i == 0 else 0 * flat) for i in range(4))
    par = {k: ops.Parameter.borrow(ctx, k, s, DeviceArray.borrow(ctx, P.ptr + 4 * offsets[k], s, owner=P),
                                   DeviceArray.borrow(ctx, G.ptr + 4 * offsets[k], s, owner=G)) for k, s in sizes.items()}
    matrices = ops.MuonMatrices(ctx, [offsets["M"]], [H], [H], [0.2 * np.sqrt(H)])
    x, y, n, dn, dy, dx = (DeviceArray(ctx, (T, H)) for _ in range(6))
    row_loss, lse, loss = DeviceArray(ctx, (T,)), DeviceArray(ctx, (T,)), DeviceArray(ctx, (1,))
    norm = DeviceArray(ctx, (4,))
    ids = r.integers(0, V, T).astype(np.int32)
    labels = np.where(r.random(T) < 0.3, r.integers(0, V, T), ops.NO_LABEL).astype(np.int32)
    dev_ids, dev_labels = DeviceArray.from_numpy(ctx, ids), DeviceArray.from_numpy(ctx, labels)
    scale = 1.0 / (labels >= 0).sum()

    # The same in 64 bits.
    q = {k: v.astype(np.float32).astype(np.float64) for k, v in p0.items()}
    mom = {k: np.zeros(s) for k, s in sizes.items()}
    var = {k: np.zeros(s) for k, s in sizes.items()}

    def reference(step):
        X = q["E"][ids]
        Y = X @ q["M"].T
        mean, rstd = Y.mean(1, keepdims=True), 1 / np.sqrt(Y.var(1, keepdims=True) + eps)
        hat = (Y - mean) * rstd
        N = hat * q["gamma"]
        z = N @ q["E"].T + q["bias"]
        lse_ = np.log(np.exp(z - z.max(1, keepdims=True)).sum(1)) + z.max(1)
        has = labels >= 0
        Gz = np.exp(z - lse_[:, None])
        Gz[np.arange(T)[has], labels[has]] -= 1
        Gz *= (has * scale)[:, None]
        value = scale * (lse_ - z[np.arange(T), np.where(has, labels, 0)])[has].sum()
        dN = Gz @ q["E"]
        g = {"E": Gz.T @ N, "bias": Gz.sum(0), "gamma": (dN * hat).sum(0)}
        t = dN * q["gamma"]
        dY = rstd * (t - t.mean(1, keepdims=True) - hat * (t * hat).mean(1, keepdims=True))
        g["M"] = dY.T @ X
        np.add.at(g["E"], ids, dY @ q["M"])
        total = np.sqrt(sum((v ** 2).sum() for v in g.values()))
        c = min(1.0, 0.5 / (total + 1e-6))
        for k in ("E", "gamma", "bias"):
            mom[k] = 0.9 * mom[k] + 0.1 * c * g[k]
            var[k] = 0.999 * var[k] + 0.001 * (c * g[k]) ** 2
            q[k] = q[k] * (1 - 1e-3 * 0.01) - 1e-3 / (1 - 0.9 ** step) * mom[k] / (
                np.sqrt(var[k]) / np.sqrt(1 - 0.999 ** step) + 1e-8)
        mom["M"] = 0.95 * mom["M"] + c * g["M"]
        q["M"] = q["M"] * (1 - lr * 0.01) - lr * 0.2 * np.sqrt(H) * _iterate(c * g["M"] + 0.95 * mom["M"], 5, np.float64)
        return value, g

    size = ctypes.c_size_t * 2
    for step in range(1, 4):
        check(L.laya_embedding_fwd(ctx.handle, dev_ids.ptr, T, par["E"].data.ptr, V, H, x.ptr, None))
        ops.linear(par["M"], None, x, T, y)
        ops.layer_norm(y, T, H, par["gamma"], None, eps, n)
        ops.vocab_ce(par["E"], par["bias"], n, dev_labels, T, row_loss, lse, scale=scale, loss=loss)
        ops.vocab_ce_backward(par["E"], par["bias"], n, dev_labels, T, lse, dn, scale=scale)
        dy.fill(0.0)
        ops.layer_norm_backward(y, T, H, par["gamma"], None, eps, dn, dy)
        ops.linear_backward(par["M"], None, x, dy, T, dx)
        ops.embedding_backward(ctx, ids, dx, H, par["E"].gradient, V)
        value, g = reference(step)
        got = {k: par[k].gradient.numpy() for k in sizes}
        for k in sizes:
            rel = np.linalg.norm(got[k] - g[k]) / np.linalg.norm(g[k])
            assert rel < 2.0 ** -15, (step, k, rel)
        assert abs(loss.numpy()[0] - value) < 2.0 ** -15 * value
        check(L.laya_grad_norm(ctx.handle, G.ptr, G.size, 0.5, norm.ptr, norm.ptr + 8))
        coef = DeviceArray.borrow(ctx, norm.ptr + 8, (1,), owner=norm)
        ops.muon(matrices, P, G, M1, learning_rate=lr, mu=0.95, weight_decay=0.01, coef=coef)
        begin, end = size(0, offsets["gamma"]), size(offsets["M"], at)
        rates = (ctypes.c_double * 2)(1e-3, 1e-3)
        check(L.laya_adamw(ctx.handle, P.ptr, G.ptr, M1.ptr, M2.ptr, 2, begin, end, rates, 0.9, 0.999, 1e-8, 0.01, step,
                           coef.ptr, 0))
        check(L.laya_fill(ctx.handle, G.ptr, 0.0, G.size))
        for k in sizes:
            now = par[k].data.numpy()
            moved = np.linalg.norm(q[k] - p0[k])
            assert np.linalg.norm(now - q[k]) < 2.0 ** -9 * moved + 2.0 ** -22 * np.linalg.norm(q[k]), (step, k)
