"""Layer normalisation, embedding lookup and distillation loss, forward and backward, against their definitions
in 64 bits (extended precision for float64 data).

Tolerances follow from the arithmetic: u is half a step of the accumulation type; a sum of terms with a chain of
at most k additions is off by at most k u sum|terms|; a product, quotient or root adds u relative, an exponential
or logarithm of the CUDA library one step (2 u); the result is rounded once, by half a step of its type.  The
chain of a row sum is at most n / 32 additions in one lane plus the folds of a block (5 in a warp, at most 32
warps)."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ["f2", "f4", "f8"]
WIDE = {"f2": np.float64, "f4": np.float64, "f8": np.longdouble}
ACC = {"f2": "f4", "f4": "f4", "f8": "f8"}


def unit(dt):
    return float(np.finfo(ACC[np.dtype(dt).str[1:]]).eps) / 2


def half_step(y, dt):
    """Half a step of type `dt` at the values y (below the normal range: half the smallest number)."""
    f = np.finfo(dt)
    return np.maximum(np.abs(y) * (float(f.eps) / 2), float(f.smallest_subnormal) / 2)


def chain(n):
    return n / 32 + 40


def close(got, want, tol, dt):
    """|got - want| <= tol + half a step, for finite values; the others equal."""
    got = np.asarray(got)
    assert got.dtype == np.dtype(dt) and got.shape == want.shape
    g = got.astype(want.dtype)
    tol = np.broadcast_to(tol, want.shape)
    top = float(np.finfo(dt).max)
    fine = np.isfinite(want) & (np.abs(want) < top)
    assert np.array_equal(np.isnan(g), np.isnan(want))
    off = np.abs(g - want)[fine]
    allowed = (tol + half_step(want, dt))[fine] * (1 + 1e-6)
    if off.size:
        worst = np.argmax(off - allowed)
        assert off[worst] <= allowed[worst], (off[worst], allowed[worst], int(np.sum(off > allowed)))
    rest = ~fine & ~np.isnan(want)
    assert np.array_equal(np.isinf(g[rest]), np.isinf(want[rest]) | (np.abs(want[rest]) >= top))


def dev(x):
    import dpnp_b200 as dp

    return dp.asarray(x)


def host(x):
    return x.asnumpy()


# ------------------------------------------------------------------------------------ layer normalisation
def norm_reference(x, w, b, eps, wide):
    n = x.shape[-1]
    x = x.astype(wide)
    m = x.mean(-1, keepdims=True)
    v = ((x - m)**2).mean(-1, keepdims=True)
    r = 1 / np.sqrt(v + wide(eps))
    h = (x - m) * r
    w = np.ones(n, wide) if w is None else w.astype(wide)
    b = np.zeros(n, wide) if b is None else b.astype(wide)
    return h * w + b, m, r, v, h, w, b


def check_norm(x, w, b, eps, y, mean, rstd):
    dt = x.dtype.str[1:]
    wide, u, k = WIDE[dt], unit(dt), chain(x.shape[-1])
    # eps reaches the kernel in the accumulation type
    want, m, r, v, h, ww, bb = norm_reference(x, w, b, np.dtype(ACC[dt]).type(eps), wide)
    off_m = (k + 2) * u * np.abs(x.astype(wide)).mean(-1, keepdims=True)
    e = np.maximum(v + eps, np.finfo(ACC[dt]).tiny)
    rel_r = ((k + 6) * u + off_m**2 / e) / 2 + 3 * u
    close(mean, m[..., 0], off_m[..., 0], ACC[dt])
    close(rstd, r[..., 0], (r * rel_r)[..., 0], ACC[dt])
    tol = np.abs(ww) * (r * off_m + np.abs(h) * (rel_r + 3 * u)) + 3 * u * (np.abs(h * ww) + np.abs(bb))
    close(y, want, tol, dt)


NORM_TYPES = [("f2", "f2"), ("f2", "f4"), ("f4", "f4"), ("f8", "f8")]
WIDTHS = [1, 2, 3, 7, 8, 31, 33, 64, 100, 127, 257, 512, 1000, 1023, 1024, 1025, 1537, 2048, 4096, 5000, 8191, 16384,
          20001, 40000, 70001]


def norm_data(rows, n, dt, wt, seed):
    rng = np.random.default_rng(seed)
    x = (rng.normal(0, 1, (rows, n)) * np.exp(rng.normal(0, 1, (rows, 1))) + rng.normal(0, 3, (rows, 1))).astype(dt)
    return x, (1 + 0.3 * rng.normal(0, 1, n)).astype(wt), (0.3 * rng.normal(0, 1, n)).astype(wt), rng


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("dt,wt", NORM_TYPES)
def test_layer_norm(n, dt, wt):
    import dpnp_b200 as dp

    for rows in (1, 5, 37):
        x, w, b, _ = norm_data(rows, n, dt, wt, n + rows)
        y, mean, rstd = dp.layer_norm(dev(x), dev(w), dev(b), eps=1e-5, return_stats=True)
        check_norm(x, w, b, 1e-5, host(y), host(mean), host(rstd))
    again = dp.layer_norm(dev(x), dev(w), dev(b), eps=1e-5)
    assert np.array_equal(host(again), host(y))
    y, mean, rstd = dp.layer_norm(dev(x), eps=0.25, return_stats=True)
    check_norm(x, None, None, 0.25, host(y), host(mean), host(rstd))
    y, mean, rstd = dp.layer_norm(dev(x), None, dev(b), return_stats=True)
    check_norm(x, None, b, 1e-5, host(y), host(mean), host(rstd))


@pytest.mark.parametrize("dt,wt", NORM_TYPES)
def test_layer_norm_many_rows(dt, wt):
    import dpnp_b200 as dp

    for rows, n in ((3000, 96), (1500, 769), (700, 2048), (401, 4097)):
        x, w, b, _ = norm_data(rows, n, dt, wt, rows)
        y, mean, rstd = dp.layer_norm(dev(x), dev(w), dev(b), return_stats=True)
        check_norm(x, w, b, 1e-5, host(y), host(mean), host(rstd))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,n,pad", [(2, 37, 1), (9, 37, 0), (1183, 37, 0), (1200, 300, 5), (2500, 301, 1), (1300, 2049, 0),
                                        (297, 4095, 2), (600, 8191, 1), (593, 130, 0), (1000, 5, 3)])
def test_layer_norm_rows_off_the_vector_grid(dt, rows, n, pad):
    """Odd widths and padded rows, row counts around the numbers of blocks; x, dy and the results start at different
    places within 16 bytes."""
    import dpnp_b200 as dp

    if rows * n > 2e6 and dt == "f8":
        rows //= 3
    x, w, b, rng = norm_data(rows, n + pad, dt, dt, rows + n)
    w, b, dy = w[:n], b[:n], rng.normal(0, 1, (rows, n)).astype(dt)
    d = dev(x)[:, pad // 2:pad // 2 + n]
    x = np.ascontiguousarray(x[:, pad // 2:pad // 2 + n])
    y, mean, rstd = dp.layer_norm(d, dev(w), dev(b), return_stats=True)
    check_norm(x, w, b, 1e-5, host(y), host(mean), host(rstd))
    out = dp.layer_norm_backward(dev(dy), d, mean, rstd, dev(w))
    check_norm_backward(x, dy, w, host(mean), host(rstd), *map(host, out))
    buf = dp.zeros(rows * n + 8, dtype=dt)
    shifted = buf[3:rows * n + 3].reshape(rows, n)
    shifted[:] = dev(dy)
    out = dp.layer_norm_backward(shifted, d, mean, rstd, dev(w))
    check_norm_backward(x, dy, w, host(mean), host(rstd), *map(host, out))
    target = buf[1:rows * n + 1].reshape(rows, n)
    dp.layer_norm(d, dev(w), dev(b), out=target)
    check_norm(x, w, b, 1e-5, host(target), host(mean), host(rstd))
    assert not host(buf)[:1].any() and not host(buf)[rows * n + 4:].any()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,n,pad", [(2600, 523, 0), (2600, 305, 2), (2600, 151, 1), (900, 4099, 0), (601, 9001, 0), (450, 12003, 1),
                                        (301, 16001, 3), (160, 32011, 0)])
def test_layer_norm_rows_off_the_vector_grid_in_other_forms(dt, rows, n, pad):
    """The widths at which the forward kernel's threads, accesses and places of the weights change."""
    test_layer_norm_rows_off_the_vector_grid(dt, rows, n, pad)


def check_norm_backward(x, dy, w, mean, rstd, dx, dw, db):
    dt = x.dtype.str[1:]
    wide, u, n = WIDE[dt], unit(dt), x.shape[-1]
    k, kr = chain(n), int(np.prod(x.shape[:-1])) + 8
    lead = tuple(range(x.ndim - 1))
    r = rstd.astype(wide)[..., None]
    h = (x.astype(wide) - mean.astype(wide)[..., None]) * r
    g = dy.astype(wide)
    a = g if w is None else g * w.astype(wide)
    c1, c2 = a.mean(-1, keepdims=True), (a * h).mean(-1, keepdims=True)
    want = r * (a - c1 - h * c2)
    off1 = (k + 3) * u * np.abs(a).mean(-1, keepdims=True)
    off2 = (k + 6) * u * np.abs(a * h).mean(-1, keepdims=True)
    tol = np.abs(r) * (off1 + np.abs(h) * off2 + 5 * u * (np.abs(a) + np.abs(c1) + np.abs(h * c2))) + 2 * u * np.abs(want)
    close(dx, want, tol, dt)
    if dw is not None:
        # a product h of two roundings, one product and a chain of at most one addition a row
        close(dw, (g * h).sum(lead), (kr + 5) * u * np.abs(g * h).sum(lead), dw.dtype.str[1:])
        close(db, g.sum(lead), (kr + 2) * u * np.abs(g).sum(lead), db.dtype.str[1:])


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("dt,wt", NORM_TYPES)
def test_layer_norm_backward(n, dt, wt):
    import dpnp_b200 as dp

    for rows in (1, 6, 41):
        x, w, b, rng = norm_data(rows, n, dt, wt, n + rows)
        dy = rng.normal(0, 1, x.shape).astype(dt)
        _, mean, rstd = dp.layer_norm(dev(x), dev(w), dev(b), return_stats=True)
        m, r = host(mean), host(rstd)
        dx, dw, db = dp.layer_norm_backward(dev(dy), dev(x), mean, rstd, dev(w))
        check_norm_backward(x, dy, w, m, r, host(dx), host(dw), host(db))
        again = dp.layer_norm_backward(dev(dy), dev(x), mean, rstd, dev(w))
        assert all(np.array_equal(host(p), host(q)) for p, q in zip(again, (dx, dw, db)))
    dx, dw, db = dp.layer_norm_backward(dev(dy), dev(x), mean, rstd)
    assert dw.dtype == np.dtype(dt)
    check_norm_backward(x, dy, None, m, r, host(dx), host(dw), host(db))
    dx, none1, none2 = dp.layer_norm_backward(dev(dy), dev(x), mean, rstd, dev(w), weight_grads=False)
    assert none1 is None and none2 is None
    check_norm_backward(x, dy, w, m, r, host(dx), None, None)


@pytest.mark.parametrize("dt,wt", NORM_TYPES)
def test_layer_norm_backward_many_rows(dt, wt):
    import dpnp_b200 as dp

    for rows, n in ((5000, 40), (3001, 768), (1200, 1023), (900, 4096), (333, 12001)):
        x, w, b, rng = norm_data(rows, n, dt, wt, rows)
        dy = rng.normal(0, 1, x.shape).astype(dt)
        _, mean, rstd = dp.layer_norm(dev(x), dev(w), dev(b), return_stats=True)
        out = dp.layer_norm_backward(dev(dy), dev(x), mean, rstd, dev(w))
        check_norm_backward(x, dy, w, host(mean), host(rstd), *map(host, out))


def test_layer_norm_gradient_against_differences():
    """float64: the directional derivative of sum(g * y) by a central difference.  With a step of 1e-5 its error is
    1e-10 of the third derivative (of the order of the function's size here) plus 1e-16 / 1e-5 of the sum."""
    import dpnp_b200 as dp

    x, w, b, rng = norm_data(7, 65, "f8", "f8", 3)
    g = rng.normal(0, 1, x.shape)
    _, mean, rstd = dp.layer_norm(dev(x), dev(w), dev(b), return_stats=True)
    grads = [host(t) for t in dp.layer_norm_backward(dev(g), dev(x), mean, rstd, dev(w))]

    def loss(x_, w_, b_):
        return float(np.sum(g * host(dp.layer_norm(dev(x_), dev(w_), dev(b_)))))

    base = [x, w, b]
    for i in range(3):
        d = rng.normal(0, 1, base[i].shape)
        at = [[p + (s * 1e-5 * d if j == i else 0) for j, p in enumerate(base)] for s in (1, -1)]
        assert abs((loss(*at[0]) - loss(*at[1])) / 2e-5 - float(np.sum(grads[i] * d))) < 1e-6 * np.sum(np.abs(g))


@pytest.mark.parametrize("dt", TYPES)
def test_layer_norm_layouts(dt):
    """Slices, broadcasts, reversed and transposed operands give what their contiguous copies give."""
    import dpnp_b200 as dp

    rng = np.random.default_rng(5)
    base = rng.normal(0, 1, (6, 10, 131)).astype(dt)
    d = dev(base)
    w = rng.normal(1, 0.1, 131).astype(dt)
    views = [(d[:, :, 1:], base[:, :, 1:]), (d[::-1], base[::-1]), (d[:, 2:7], base[:, 2:7]), (d[:, ::3, :128], base[:, ::3, :128]),
             (d[:, -1], base[:, -1]), (d.transpose(1, 0, 2), base.transpose(1, 0, 2)), (d[:, :, ::2], base[:, :, ::2]),
             (dp.broadcast_to(d[0, :1], (10, 131)), np.broadcast_to(base[0, :1], (10, 131))), (d[0, 0], base[0, 0])]
    for v, b in views:
        n = b.shape[-1]
        y, mean, rstd = dp.layer_norm(v, dev(w[:n]), return_stats=True)
        dy = rng.normal(0, 1, b.shape).astype(dt)
        check_norm(np.ascontiguousarray(b), w[:n], None, 1e-5, host(y), host(mean), host(rstd))
        out = dp.layer_norm_backward(dev(dy), v, mean, rstd, dev(w[:n]))
        check_norm_backward(np.ascontiguousarray(b), dy, w[:n], host(mean), host(rstd), *map(host, out))
    wide = dev(np.zeros(262, dt))
    wide[::2] = dev(w)
    y = dp.layer_norm(d, wide[::2])                                  # a strided weight
    assert np.array_equal(host(y), host(dp.layer_norm(d, dev(w))))


@pytest.mark.parametrize("axis", [0, 1, -1, (1, 2), (2, 0), (0, 1, 2)])
def test_layer_norm_axes(axis):
    import dpnp_b200 as dp

    rng = np.random.default_rng(6)
    x = rng.normal(0, 2, (5, 12, 9)).astype("f4")
    axes = axis if isinstance(axis, tuple) else (axis,)
    axes = tuple(a % 3 for a in axes)
    shape = tuple(x.shape[a] for a in axes)
    w, b = rng.normal(1, 0.2, shape).astype("f4"), rng.normal(0, 0.2, shape).astype("f4")
    perm = [i for i in range(3) if i not in axes] + list(axes)
    rest = tuple(x.shape[i] for i in perm[:3 - len(axes)])
    moved = np.ascontiguousarray(x.transpose(perm)).reshape(rest + (-1,))
    y, mean, rstd = dp.layer_norm(dev(x), dev(w), dev(b), axis=axis, return_stats=True)
    assert y.shape == x.shape and mean.shape == rest
    check_norm(moved, w.ravel(), b.ravel(), 1e-5, host(y).transpose(perm).reshape(moved.shape), host(mean), host(rstd))
    dy = rng.normal(0, 1, x.shape).astype("f4")
    dx, dw, db = dp.layer_norm_backward(dev(dy), dev(x), mean, rstd, dev(w), axis=axis)
    assert dx.shape == x.shape and dw.shape == shape
    check_norm_backward(moved, np.ascontiguousarray(dy.transpose(perm)).reshape(moved.shape), w.ravel(), host(mean),
                        host(rstd), host(dx).transpose(perm).reshape(moved.shape), host(dw).ravel(), host(db).ravel())
    o = dp.empty(x.shape, dtype="f4")
    assert dp.layer_norm(dev(x), dev(w), dev(b), axis=axis, out=o) is o and np.array_equal(host(o), host(y))
    d = dev(x)
    assert np.array_equal(host(dp.layer_norm(d, dev(w), dev(b), axis=axis, out=d)), host(y))


@pytest.mark.parametrize("n", [100, 1537, 4096, 70001])
@pytest.mark.parametrize("dt", TYPES)
def test_layer_norm_out_and_in_place(dt, n):
    import dpnp_b200 as dp

    x, w, b, rng = norm_data(11, n, dt, dt, n)
    dy = rng.normal(0, 1, x.shape).astype(dt)
    y, mean, rstd = dp.layer_norm(dev(x), dev(w), dev(b), return_stats=True)
    big = dp.zeros((11, n + 5), dtype=dt)
    m2, r2 = dp.empty(11, dtype=ACC[dt]), dp.empty(11, dtype=ACC[dt])
    res = dp.layer_norm(dev(x), dev(w), dev(b), return_stats=True, out=(big[:, 3:n + 3], m2, r2))
    # rows that start elsewhere may be read in narrower accesses, and the sums then run in another order
    assert res[1] is m2
    check_norm(x, w, b, 1e-5, host(big)[:, 3:n + 3], host(m2), host(r2))
    assert not host(big)[:, :3].any() and not host(big)[:, n + 3:].any()
    d = dev(x)
    assert dp.layer_norm(d, dev(w), dev(b), out=d) is d and np.array_equal(host(d), host(y))
    d = dev(np.concatenate([x.ravel(), x.ravel()[:1]]))               # shifted by one element: a partial overlap
    dp.layer_norm(d[:-1].reshape(11, n), dev(w), dev(b), out=d[1:].reshape(11, n))
    check_norm(x, w, b, 1e-5, host(d)[1:].reshape(11, n), host(mean), host(rstd))
    want = [host(t) for t in dp.layer_norm_backward(dev(dy), dev(x), mean, rstd, dev(w))]
    for over in (0, 1):
        p = [dev(dy), dev(x)]
        res = dp.layer_norm_backward(p[0], p[1], mean, rstd, dev(w), out=(p[over], None, None))
        assert res[0] is p[over] and all(np.array_equal(host(r), v) for r, v in zip(res, want))
    strided = dp.zeros((n, 2), dtype=dt)
    with pytest.raises(ValueError):               # results in one range of memory, though not in the same places
        dp.layer_norm_backward(dev(dy), dev(x), mean, rstd, dev(w), out=(None, strided[:, 0], strided[:, 1]))
    other = dp.zeros((n, 2), dtype=dt)
    dp.layer_norm_backward(dev(dy), dev(x), mean, rstd, dev(w), out=(None, strided[:, 0], other[:, 1]))
    assert np.array_equal(host(strided)[:, 0], want[1]) and np.array_equal(host(other)[:, 1], want[2])
    assert not host(strided)[:, 1].any() and not host(other)[:, 0].any()
    wt = dev(w)
    assert np.array_equal(host(dp.layer_norm_backward(dev(dy), dev(x), mean, rstd, wt, out=(None, wt, None))[1]), want[1])


@pytest.mark.parametrize("n", [5, 300, 4096, 33000, 70000])
def test_layer_norm_values(n):
    import dpnp_b200 as dp

    x = np.random.default_rng(n).normal(0, 1, (8, n)).astype("f4")
    x[1] = 7.25                                    # no variance: h is 0 up to the mean's rounding
    x[2] += 1e4                                    # far from zero
    x[3, n // 2] = np.nan
    x[4, 0] = np.inf
    x[5] *= 1e18                                   # squares still within float32
    x[6] = 0
    y, mean, rstd = dp.layer_norm(dev(x), return_stats=True)
    y, m, r = host(y), host(mean), host(rstd)
    fine = [0, 1, 2, 5, 6, 7]
    check_norm(x[fine], None, None, 1e-5, y[fine], m[fine], r[fine])
    assert np.isnan(y[3]).all() and np.isnan(y[4]).all() and not y[6].any()
    dy = np.ones_like(x)
    dx, dw, db = dp.layer_norm_backward(dev(dy[fine]), dev(x[fine]), dev(m[fine]), dev(r[fine]))
    check_norm_backward(x[fine], dy[fine], None, m[fine], r[fine], host(dx), host(dw), host(db))
    h = np.full((2, n), 60000, "f2")               # a sum far above float16's range
    assert not np.isnan(host(dp.layer_norm(dev(h)))).any() and abs(float(host(dp.mean(dev(h.astype("f4"))))) - 60000) < 60


def test_layer_norm_empty():
    import dpnp_b200 as dp

    y, mean, rstd = dp.layer_norm(dp.zeros((0, 8), dtype="f4"), return_stats=True)
    assert y.shape == (0, 8) and mean.shape == (0,)
    dx, dw, db = dp.layer_norm_backward(y, y, mean, rstd)
    assert dx.shape == (0, 8) and not host(dw).any() and not host(db).any() and dw.shape == (8,)


# ---------------------------------------------------------------------------------------------- embedding
IDS = ["i4", "i8", "i2", "u1", "u8"]


@pytest.mark.parametrize("n", [1, 2, 3, 8, 17, 64, 129, 768, 1000, 4096, 5001])
@pytest.mark.parametrize("dt", TYPES)
def test_embedding(n, dt):
    import dpnp_b200 as dp

    rng = np.random.default_rng(n)
    table = rng.normal(0, 1, (130, n)).astype(dt)
    for shape in ((), (1,), (3, 5), (2, 3, 40)):
        ids = rng.integers(-3, 134, shape).astype("i4")
        for scale in (1.0, 0.3, 22.627416997969522):
            got = host(dp.embedding(dev(table), dev(ids), scale=scale))
            acc = np.dtype(ACC[dt]).type
            want = np.zeros(shape + (n,), dt)
            known = (ids >= 0) & (ids < 130)
            want[known] = (table[ids[known]].astype(ACC[dt]) * acc(scale)).astype(dt)
            assert got.dtype == table.dtype and np.array_equal(got, want)


@pytest.mark.parametrize("idt", IDS)
def test_embedding_index_types_and_layouts(idt):
    import dpnp_b200 as dp

    rng = np.random.default_rng(1)
    table = rng.normal(0, 1, (100, 48)).astype("f4")
    ids = rng.integers(0, 100, (12, 10)).astype(idt)
    d, i = dev(table), dev(ids)
    assert np.array_equal(host(dp.embedding(d, i.T)), table[ids.T.astype(int)])
    assert np.array_equal(host(dp.embedding(d[:, 1:47], i[::2, ::3])), table[:, 1:47][ids[::2, ::3].astype(int)])
    assert np.array_equal(host(dp.embedding(d[::-1], i)), table[::-1][ids.astype(int)])
    assert np.array_equal(host(dp.embedding(d.T, dev(np.arange(48).astype(idt)))), table.T)
    assert np.array_equal(host(dp.embedding(dp.broadcast_to(d[5], (100, 48)), i)), np.broadcast_to(table[5], (12, 10, 48)))
    big = dp.zeros((12, 10, 50), dtype="f4")
    dp.embedding(d, i, out=big[:, :, 1:49])
    want = np.zeros((12, 10, 50), "f4")
    want[:, :, 1:49] = table[ids.astype(int)]
    assert np.array_equal(host(big), want)
    over = dev(table)                                                 # the result on top of the table
    dp.embedding(over, i[0], out=over[:10])
    assert np.array_equal(host(over)[:10], table[ids[0].astype(int)]) and np.array_equal(host(over)[10:], table[10:])


def test_embedding_extreme_ids():
    import dpnp_b200 as dp

    table = np.arange(12, dtype="f4").reshape(4, 3) + 1
    ids = np.array([0, 3, 4, -1, 2**31 - 1, -2**31, 2**40, -2**63, 2**63 - 1, 2**32], "i8")
    got = host(dp.embedding(dev(table), dev(ids)))
    assert np.array_equal(got[:2], table[[0, 3]]) and not got[2:].any()
    g = host(dp.embedding_backward(dev(np.ones((10, 3), "f4")), dev(ids), 4))
    assert np.array_equal(g, np.array([[1, 1, 1], [0, 0, 0], [0, 0, 0], [1, 1, 1]], "f4"))
    u = np.array([0, 2**63, 2**64 - 1], "u8")
    assert np.array_equal(host(dp.embedding(dev(table), dev(u)))[:, 0], [1, 0, 0])
    nan = np.full((4, 3), np.nan, "f4")
    assert not host(dp.embedding(dev(nan), dev(np.array([-1, 9])))).any()
    empty = dp.embedding(dp.zeros((0, 3), dtype="f4"), dev(ids))
    assert empty.shape == (10, 3) and not host(empty).any()


def check_embedding_backward(dout, ids, rows, scale, got, gt):
    dt = dout.dtype.str[1:]
    wide, u = WIDE[dt], unit(dt)
    flat, g = ids.ravel().astype("i8"), dout.reshape(-1, dout.shape[-1]).astype(wide)
    known = (flat >= 0) & (flat < rows)
    want, mag = np.zeros((rows, g.shape[1]), wide), np.zeros((rows, g.shape[1]), wide)
    np.add.at(want, flat[known], g[known])
    np.add.at(mag, flat[known], np.abs(g[known]))
    count = np.bincount(flat[known], minlength=rows)[:, None]
    s = wide(np.dtype(ACC[dt]).type(scale))
    close(got, want * s, np.abs(s) * (count + 1) * u * mag, gt)


@pytest.mark.parametrize("tokens", [1, 2, 31, 128, 129, 400, 4096, 4097, 9000])
@pytest.mark.parametrize("dt,gt", [("f2", "f2"), ("f2", "f4"), ("f4", "f4"), ("f8", "f8")])
def test_embedding_backward(tokens, dt, gt):
    import dpnp_b200 as dp

    rng = np.random.default_rng(tokens)
    for rows, n, skew in ((1, 40, 1), (7, 17, 1), (500, 64, 3), (3000, 129, 6), (70000, 8, 2)):
        ids = (rows * rng.uniform(0, 1, tokens)**skew).astype("i8")
        ids[rng.uniform(0, 1, tokens) < 0.05] = -1
        dout = rng.normal(0, 1, (tokens, n)).astype(dt)
        got = dp.embedding_backward(dev(dout), dev(ids), rows, scale=0.75, dtype=gt)
        check_embedding_backward(dout, ids, rows, 0.75, host(got), gt)
        again = dp.empty((rows, n), dtype=gt)
        assert dp.embedding_backward(dev(dout), dev(ids.astype("i4")), rows, scale=0.75, out=again) is again
        assert np.array_equal(host(again), host(got))


@pytest.mark.parametrize("kind", ["one row", "two rows", "all padding", "sorted", "reversed", "runs at chunk borders"])
def test_embedding_backward_distributions(kind):
    import dpnp_b200 as dp

    rng = np.random.default_rng(2)
    tokens, rows, n = 5003, 300, 96
    ids = {"one row": np.full(tokens, 17), "two rows": rng.integers(0, 2, tokens) * 299, "all padding": np.full(tokens, -1),
           "sorted": np.sort(rng.integers(0, rows, tokens)), "reversed": np.sort(rng.integers(0, rows, tokens))[::-1],
           "runs at chunk borders": np.minimum(np.arange(tokens) // 128, rows - 1)}[kind].astype("i4")
    dout = rng.normal(0, 1, (tokens, n)).astype("f4")
    got = host(dp.embedding_backward(dev(dout), dev(ids), rows))
    check_embedding_backward(dout, ids, rows, 1.0, got, "f4")


@pytest.mark.parametrize("tokens,rows,n,idt", [(140000, 1000, 24, "i4"), (70000, 300000, 4, "i8"), (1500, 600000, 3, "i4"),
                                               (131073, 5, 8, "i8"), (90000, 40, 2050, "i4")])
def test_embedding_backward_long_batches(tokens, rows, n, idt):
    """Several tiles of the sort and more than the tiles that are placed without a scan; tables of one to three digits;
    long chunks, and ids that span hundreds of them."""
    import dpnp_b200 as dp

    rng = np.random.default_rng(tokens)
    ids = (rows * rng.uniform(0, 1, tokens)**4).astype(idt)
    ids[rng.uniform(0, 1, tokens) < 0.3] = rows // 2
    ids[rng.uniform(0, 1, tokens) < 0.02] = -7
    dout = rng.normal(0, 1, (tokens, n)).astype("f4" if n > 1000 else "f8")
    got = dp.embedding_backward(dev(dout), dev(ids), rows, scale=2.0)
    check_embedding_backward(dout, ids, rows, 2.0, host(got), dout.dtype.str[1:])
    again = dp.embedding_backward(dev(dout), dev(ids), rows, scale=2.0)
    assert np.array_equal(host(again), host(got))


@pytest.mark.parametrize("n", [5000, 20011])
@pytest.mark.parametrize("dt", ["f2", "f4"])
def test_embedding_backward_frequent_ids_of_wide_rows(dt, n):
    """Runs over several chunks, in rows of several blocks."""
    import dpnp_b200 as dp

    rng = np.random.default_rng(n)
    ids = np.where(rng.uniform(0, 1, 400) < 0.6, 3, rng.integers(-1, 6, 400)).astype("i4")
    dout = rng.normal(0, 1, (400, n)).astype(dt)
    check_embedding_backward(dout, ids, 7, 0.5, host(dp.embedding_backward(dev(dout), dev(ids), 7, scale=0.5)), dt)


def test_embedding_backward_layouts():
    import dpnp_b200 as dp

    rng = np.random.default_rng(3)
    dout = rng.normal(0, 1, (20, 30, 70)).astype("f4")
    ids = rng.integers(-1, 60, (20, 30)).astype("i4")
    d, i = dev(dout), dev(ids)
    for v, iv, b, ib in ((d[:, :, 3:], i, dout[:, :, 3:], ids), (d[::2, 5:], i[::2, 5:], dout[::2, 5:], ids[::2, 5:]),
                         (d.transpose(1, 0, 2), i.T, dout.transpose(1, 0, 2), ids.T), (d[:, :, ::2], i, dout[:, :, ::2], ids),
                         (dp.broadcast_to(d[0, 0], (20, 30, 70)), i, np.broadcast_to(dout[0, 0], (20, 30, 70)), ids)):
        got = host(dp.embedding_backward(v, iv, 60))
        check_embedding_backward(np.ascontiguousarray(b), np.ascontiguousarray(ib), 60, 1.0, got, "f4")
    big = dp.full((60, 75), 7, dtype="f4")
    dp.embedding_backward(d, i, 60, out=big[:, 2:72])
    check_embedding_backward(dout, ids, 60, 1.0, host(big)[:, 2:72], "f4")
    assert (host(big)[:, :2] == 7).all() and (host(big)[:, 72:] == 7).all()
    none = dp.embedding_backward(d[:0], i[:0], 60)
    assert none.shape == (60, 70) and not host(none).any()
    assert dp.embedding_backward(d, i, 0).shape == (0, 70)


# ------------------------------------------------------------------------------------------- distillation
def distil_reference(z, t, idx, temp, wide):
    """loss, gradient for dloss = 1, statistics, and the pieces that the tolerances need."""
    z, t = z.astype(wide), t.astype(wide)
    v = z.shape[-1]
    idx = idx.astype("i8")
    counts = (idx >= 0) & (idx < v) & (t != -np.inf)          # a NaN counts
    used = counts.any(-1)
    with np.errstate(all="ignore"):
        tt = np.where(counts, t, -np.inf)
        top = tt.max(-1, keepdims=True, initial=-np.inf)
        e = np.where(counts, np.exp((tt - top) / temp), 0)
        s = e.sum(-1, keepdims=True)
        p = np.where(counts, e / s, 0)
        logp = np.where(counts, (tt - top) / temp - np.log(s), 0)
        m = z.max(-1, keepdims=True)
        masked = z == -np.inf
        d = np.where(masked, -np.inf, (z - m) / temp)
        ls = np.log(np.exp(d).sum(-1, keepdims=True))
        q = np.where(masked, 0, np.exp(d - ls))
        at = np.take_along_axis(d, np.where(counts, idx, 0), -1)
        logq = np.where(np.take_along_axis(masked, np.where(counts, idx, 0), -1), -np.inf, at - ls)
        terms = np.where(p != 0, p * (logp - logq), 0)
        loss = np.where(used, temp**2 * terms.sum(-1), 0)
        w = np.zeros_like(z)
        np.add.at(w, tuple(np.indices(idx.shape)[:-1]) + (np.where(counts, idx, 0),), p)
        grad = np.where(used[..., None], temp * (q - w), 0)
        stats = np.where(used[..., None], np.concatenate([m, ls], -1), 0)
    return loss, grad, stats, dict(p=p, logp=logp, logq=logq, q=q, w=w, d=d, at=at, tt=tt, top=top, used=used, counts=counts)


def check_distil(z, t, idx, temp, loss=None, grad=None, stats=None, dloss=1.0):
    dt = z.dtype.str[1:]
    wide, u, acc = WIDE[dt], unit(dt), ACC[dt]
    temp = wide(np.dtype(acc).type(temp))
    want_loss, want_grad, want_stats, c = distil_reference(z, t, idx, temp, wide)
    v, k = z.shape[-1], t.shape[-1]
    with np.errstate(all="ignore"):
        # exponents: a difference, the reciprocal of T and a product, 3 u relative; exp and log one step
        d = np.where(np.isfinite(c["d"]), np.abs(c["d"]), 0)
        # the sum's chain: at most V / 256 additions in a lane and the folds, each with one rescaling (an
        # exponential of a difference and a product) at most: 4 roundings and 3 u of the exponent
        rel_s = (4 * (v / 256 + 64)) * u + 6 * u * np.max(d * (c["q"] > 0), -1, keepdims=True)
        ls = np.abs(np.where(np.isfinite(want_stats[..., 1:]), want_stats[..., 1:], 0))
        off_ls = rel_s + 2 * u * ls
        dt_ = np.where(c["counts"], np.abs(c["tt"] - c["top"]) / temp, 0)
        dt_ = np.where(np.isfinite(dt_), dt_, 0)
        rel_p = 3 * u * dt_ + (k + 8) * u + 3 * u * np.max(dt_, -1, keepdims=True, initial=0)
        off_logp = 3 * u * dt_ + (k + 8) * u + 3 * u * np.max(dt_, -1, keepdims=True, initial=0) + 2 * u * np.abs(c["logp"])
        at = np.where(np.isfinite(c["at"]), np.abs(c["at"]), 0)
        logq = np.where(np.isfinite(c["logq"]), np.abs(c["logq"]), 0)
        off_logq = 3 * u * at + off_ls + 2 * u * logq
        terms = np.abs(np.where(np.isfinite(c["logq"]) & (c["p"] > 0), c["p"] * (c["logp"] - c["logq"]), 0))
        if loss is not None:
            tol = temp**2 * ((np.where(c["p"] > 0, c["p"], 0) * (off_logp + off_logq)).sum(-1)
                             + ((rel_p + (k + 8) * u) * terms).sum(-1))
            close(loss, want_loss, np.where(np.isfinite(tol), tol, 0), acc)
        if stats is not None:
            assert np.array_equal(np.asarray(stats)[..., 0].astype(wide), want_stats[..., 0], equal_nan=True)
            close(np.asarray(stats)[..., 1], want_stats[..., 1], np.where(c["used"], off_ls[..., 0], 0), acc)
        if grad is not None:
            g = np.asarray(dloss, wide)
            g = g[..., None] if g.ndim else g
            rel_q = 3 * u * d + off_ls + u * (d + ls) + 4 * u
            off_w = np.zeros_like(c["w"])
            idx = idx.astype("i8")
            np.add.at(off_w, tuple(np.indices(idx.shape)[:-1]) + (np.where(c["counts"], idx, 0),), c["p"] * rel_p)
            tol = np.abs(g) * temp * (c["q"] * rel_q + off_w + (k + 4) * u * c["w"] + 4 * u * (c["q"] + c["w"]))
            # below the normal range of the accumulation type a rounding is off by half the smallest number s, not
            # by u relative: the exponential by s, then two products with T g and the quotient p by s / 2 each,
            # the earlier ones scaled by the later factors
            tol = tol + 2.5 * float(np.finfo(acc).smallest_subnormal) * np.maximum(1, np.abs(g) * temp)
            close(grad, want_grad * g, np.where(np.isfinite(tol), tol, 0), dt)


def distil_data(rows, vocab, k, dt, seed, idt="i4"):
    rng = np.random.default_rng(seed)
    z = rng.normal(0, 2.5, (rows, vocab)).astype(dt)
    t = rng.normal(0, 3, (rows, k)).astype(ACC[dt])
    idx = rng.integers(0, vocab, (rows, k)).astype(idt)          # some columns twice
    short = rng.uniform(0, 1, (rows, k)) < 0.1
    idx[short] = -1
    if rows > 3:
        idx[2] = -1                                              # a row without a teacher
        idx[3] = idx[3, :1] if k else idx[3]                     # one column k times
    return z, t, idx, rng


def run_distil(z, t, idx, temp, dloss=None):
    import dpnp_b200 as dp

    loss, stats = dp.distillation_loss(dev(z), dev(t), dev(idx), temperature=temp, return_stats=True)
    g = 1.0 if dloss is None else dev(dloss)
    grad = dp.distillation_loss_backward(g, dev(z), dev(t), dev(idx), stats, temperature=temp)
    check_distil(z, t, idx, temp, host(loss), None, host(stats))
    check_distil(z, t, idx, temp, None, host(grad), None, 1.0 if dloss is None else dloss)
    loss2, grad2 = dp.distillation_loss_and_grad(dev(z), dev(t), dev(idx), g, temperature=temp)
    check_distil(z, t, idx, temp, host(loss2), host(grad2), None, 1.0 if dloss is None else dloss)
    return host(loss), host(grad), host(stats)


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 33, 255, 256, 1000, 1025, 4099, 8192, 32001, 50257])
@pytest.mark.parametrize("dt", TYPES)
def test_distillation(vocab, dt):
    for rows, k, temp in ((1, 1, 1.0), (6, 8, 2.0), (9, 33, 0.7)):
        z, t, idx, rng = distil_data(rows, vocab, k, dt, vocab + rows)
        run_distil(z, t, idx, temp, (rng.uniform(0.5, 2, rows) * (64 if dt == "f2" else 1)).astype(ACC[dt]))
        run_distil(z, t, idx, temp)


@pytest.mark.parametrize("dt", TYPES)
def test_distillation_many_rows_and_long_rows(dt):
    for rows, vocab, k in ((1500, 1003, 16), (700, 5000, 5), (3, 200003, 100), (2, 128000, 1024), (40, 130000, 64)):
        if rows * vocab > 2e6 and dt == "f8":
            rows = min(rows, 8)
        z, t, idx, rng = distil_data(rows, vocab, k, dt, vocab)
        run_distil(z, t, idx, 1.5, rng.uniform(0.5, 2, rows).astype(ACC[dt]))


@pytest.mark.parametrize("temp", [1e-10, 1e-6, 1e-4, 5.6e-3, 6e-3, 100.0, 1e6])
@pytest.mark.parametrize("dt", TYPES)
def test_distillation_temperatures(dt, temp):
    """Far from 1, with small logits and with ones near the end of float16."""
    for rows, vocab, scale in ((7, 1003, 1.0), (5, 1000, 6000.0), (2, 40000, 4000.0)):
        z, t, idx, rng = distil_data(rows, vocab, 9, dt, vocab)
        run_distil((z * scale).astype(dt), t, idx, temp, rng.uniform(0.5, 2, rows).astype(ACC[dt]))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("idt", IDS)
def test_distillation_types_and_shapes(dt, idt):
    import dpnp_b200 as dp

    rng = np.random.default_rng(4)
    z = rng.normal(0, 2, (3, 5, 200)).astype(dt)
    idx = rng.integers(0, 120, (3, 5, 6)).astype(idt)
    for tt in TYPES:
        t = rng.normal(0, 1, (3, 5, 6)).astype(tt)
        run_distil(z, t.astype(ACC[dt]), idx, 1.0)
        a = host(dp.distillation_loss(dev(z), dev(t), dev(idx)))
        assert np.array_equal(a, host(dp.distillation_loss(dev(z), dev(t.astype(ACC[dt])), dev(idx))))
    one = run_distil(z[0, 0], t[0, 0].astype(ACC[dt]), idx[0, 0], 1.0)
    assert one[0].shape == () and one[1].shape == (200,)


@pytest.mark.parametrize("vocab", [50, 4099, 33000])
@pytest.mark.parametrize("dt", TYPES)
def test_distillation_masks(dt, vocab):
    """Masked student logits, rows without a teacher whatever they hold, -inf and NaN entries."""
    rng = np.random.default_rng(7)
    rows, k = 14, 6
    z = rng.normal(0, 2, (rows, vocab)).astype(dt)
    t = rng.normal(0, 2, (rows, k)).astype(ACC[dt])
    idx = np.stack([rng.choice(vocab - 10, k, replace=False) for _ in range(rows)]).astype("i4")
    low = np.finfo(dt).min
    z[0, vocab - 10:] = -np.inf                     # masked columns away from the teacher's
    z[1, vocab - 10:] = low
    z[2, idx[2, 1]] = -np.inf                       # masked at a teacher's column: loss +inf
    z[3] = -np.inf                                  # everything masked
    z[4] = low                                      # everything at the lowest value: uniform
    idx[5] = -1
    z[5] = np.nan                                   # ignored row full of NaN
    idx[6] = vocab
    z[6, 0] = np.inf
    t[7] = -np.inf                                  # no teacher entry counts
    t[8, 1:] = -np.inf                              # one counts
    z[9, 3] = np.nan
    t[10, 2] = np.nan
    idx[11, 2:] = -5
    z[12, vocab - 1] = np.inf
    t[13] = [1e4, -1e4, 0, 5, 2, 1]                 # probabilities that vanish
    z[13] = z[13] * 0 + np.linspace(-30, 30, vocab).astype(dt)
    loss, grad, stats = run_distil(z, t, idx, 1.0)
    assert np.isposinf(loss[2]) and np.isposinf(loss[3]) and np.isfinite(loss[4]) and np.isnan(loss[[9, 10, 12]]).all()
    assert not loss[5:8].any() and not grad[5:8].any() and not stats[5:8].any()
    assert np.isfinite(grad[:9]).all()
    run_distil(z, t, idx, 0.5)                      # the lowest value over T = 1/2 is below the type's range
    run_distil(z, np.zeros((rows, 0), ACC[dt]), np.zeros((rows, 0), "i4"), 1.0)


@pytest.mark.parametrize("vocab", [129, 5003, 33001])
@pytest.mark.parametrize("dt", TYPES)
def test_distillation_layouts_and_in_place(dt, vocab):
    import dpnp_b200 as dp

    rng = np.random.default_rng(8)
    base = rng.normal(0, 2, (6, 4, vocab + 3)).astype(dt)
    t = rng.normal(0, 2, (6, 4, 7)).astype(ACC[dt])
    idx = rng.integers(0, vocab, (6, 4, 7)).astype("i4")
    d = dev(base)
    views = [(d[:, :, 2:vocab + 2], base[:, :, 2:vocab + 2], t, idx), (d[::-2, 1:3], base[::-2, 1:3], t[::-2, 1:3], idx[::-2, 1:3]),
             (d.transpose(1, 0, 2), base.transpose(1, 0, 2), t.transpose(1, 0, 2), idx.transpose(1, 0, 2)),
             (d[:, :, 1::2], base[:, :, 1::2], t, idx // 2)]
    for v, b, tt, ii in views:
        b = np.ascontiguousarray(b)
        loss, stats = dp.distillation_loss(v, dev(np.ascontiguousarray(tt)), dev(np.ascontiguousarray(ii)), return_stats=True)
        check_distil(b, tt, ii, 1.0, host(loss), None, host(stats))
        both = dp.distillation_loss_and_grad(v, dev(np.ascontiguousarray(tt)), dev(np.ascontiguousarray(ii)), 0.5)
        check_distil(b, tt, ii, 1.0, host(both[0]), host(both[1]), None, 0.5)
    z = np.ascontiguousarray(base[0, :, :vocab])
    tt, ii = dev(t[0]), dev(idx[0])
    loss, stats = dp.distillation_loss(dev(z), tt, ii, return_stats=True)
    want = host(dp.distillation_loss_backward(1.0, dev(z), tt, ii, stats))
    over = dev(z)
    assert dp.distillation_loss_backward(1.0, over, tt, ii, stats, out=over) is over and np.array_equal(host(over), want)
    over, first = dev(z), dp.empty(4, dtype=ACC[dt])
    res = dp.distillation_loss_and_grad(over, tt, ii, out=(first, over))
    assert res[0] is first and res[1] is over
    check_distil(z, t[0], idx[0], 1.0, host(first), host(over))
    big = dp.full((4, vocab + 9), 3, dtype=dt)
    dp.distillation_loss_backward(dev(np.asarray(1.0, ACC[dt])), dev(z), tt, ii, stats, out=big[:, 5:vocab + 5])
    assert np.array_equal(host(big)[:, 5:vocab + 5], want) and (host(big)[:, :5] == 3).all() and (host(big)[:, vocab + 5:] == 3).all()


@pytest.mark.parametrize("rows,vocab,k", [(9, 512, 300), (40, 65536, 12), (700, 32832, 40), (3, 131072, 600)])
@pytest.mark.parametrize("dt", TYPES)
def test_distillation_in_place_on_cache_lines(dt, rows, vocab, k):
    """Rows of whole lines that several blocks share, more entries than threads, rows without entries that hold NaN."""
    import dpnp_b200 as dp

    if dt == "f8":
        rows = min(rows, 12)
    z, t, idx, rng = distil_data(rows, vocab, k, dt, vocab + k)
    idx[::3] = -1
    z[::3] = np.nan
    g = rng.uniform(0.5, 2, rows).astype(ACC[dt])
    over = dev(z)
    loss, grad = dp.distillation_loss_and_grad(over, dev(t), dev(idx), dev(g), temperature=1.5, out=(None, over))
    assert grad is over
    check_distil(z, t, idx, 1.5, host(loss), host(grad), None, g)
    again = dp.distillation_loss_and_grad(dev(z), dev(t), dev(idx), dev(g), temperature=1.5)
    assert np.array_equal(host(again[0]), host(loss)) and np.array_equal(host(again[1]), host(grad))


def test_distillation_gradient_against_differences():
    """float64, central differences of the summed losses (bounds as for the layer norm)."""
    import dpnp_b200 as dp

    z, t, idx, rng = distil_data(6, 301, 9, "f8", 9)
    for temp in (1.0, 2.5):
        loss, grad = dp.distillation_loss_and_grad(dev(z), dev(t), dev(idx), temperature=temp)
        d = rng.normal(0, 1, z.shape)
        at = [float(np.sum(host(dp.distillation_loss(dev(z + s * 1e-5 * d), dev(t), dev(idx), temperature=temp)))) for s in (1, -1)]
        assert abs((at[0] - at[1]) / 2e-5 - float(np.sum(host(grad) * d))) < 1e-6 * np.sum(np.abs(d[:, :9]))


# ------------------------------------------------------------------------- together, streams and graphs
def test_a_small_language_model_trains_through_the_operators():
    """ids -> embedding -> layer norm -> logits against the tied table -> distillation loss, and back; gradients of
    both parameters against differences.  The products are broadcast products and sums of this library."""
    import dpnp_b200 as dp

    rng = np.random.default_rng(11)
    vocab, n, tokens, k, temp = 23, 12, 9, 4, 1.3
    ids = np.array([0, 3, 3, 7, 22, 3, -1, 11, 0], "i4")
    t = rng.normal(0, 2, (tokens, k))
    idx = rng.integers(0, vocab, (tokens, k)).astype("i4")
    idx[6] = -1                                                       # the padded token has no teacher
    params = [rng.normal(0, 0.5, (vocab, n)), 1 + 0.1 * rng.normal(0, 1, n), 0.1 * rng.normal(0, 1, n)]

    def forward(table, w, b):
        x = dp.embedding(table, dev(ids), scale=n**0.5)
        y, mean, rstd = dp.layer_norm(x, w, b, return_stats=True)
        logits = dp.sum(dp.multiply(y.reshape(tokens, 1, n), table.reshape(1, vocab, n)), axis=2)
        return x, y, mean, rstd, logits

    def loss_of(table, w, b):
        return float(host(dp.sum(dp.distillation_loss(forward(table, w, b)[-1], dev(t), dev(idx), temperature=temp))))

    table, w, b = map(dev, params)
    x, y, mean, rstd, logits = forward(table, w, b)
    losses, dlogits = dp.distillation_loss_and_grad(logits, dev(t), dev(idx), temperature=temp)
    dy = dp.sum(dp.multiply(dlogits.reshape(tokens, vocab, 1), table.reshape(1, vocab, n)), axis=1)
    dhead = dp.sum(dp.multiply(dlogits.reshape(tokens, vocab, 1), y.reshape(tokens, 1, n)), axis=0)
    dx, dw, db = dp.layer_norm_backward(dy, x, mean, rstd, w)
    dtable = dp.add(dhead, dp.embedding_backward(dx, dev(ids), vocab, scale=n**0.5))
    assert abs(float(host(dp.sum(losses))) - loss_of(table, w, b)) < 1e-10
    for i, g in enumerate((dtable, dw, db)):
        d = rng.normal(0, 1, params[i].shape)
        at = [loss_of(*[dev(p + (s * 1e-5 * d if j == i else 0)) for j, p in enumerate(params)]) for s in (1, -1)]
        assert abs((at[0] - at[1]) / 2e-5 - float(np.sum(host(g) * d))) < 1e-5 * (1 + np.sum(np.abs(host(g))))


def _step(dp, a):
    """One pass through every operator into the arrays of `a`."""
    dp.embedding(a["table"], a["ids"], scale=2.0, out=a["x"])
    dp.layer_norm(a["x"], a["w"], a["b"], return_stats=True, out=(a["y"], a["mean"], a["rstd"]))
    dp.distillation_loss(a["y"], a["t"], a["idx"], return_stats=True, out=(a["loss"], a["stats"]))
    dp.distillation_loss_backward(a["g"], a["y"], a["t"], a["idx"], a["stats"], out=a["dy"])
    dp.distillation_loss_and_grad(a["y"], a["t"], a["idx"], a["g"], out=(a["loss2"], a["dy2"]))
    dp.layer_norm_backward(a["dy"], a["x"], a["mean"], a["rstd"], a["w"], out=(a["dx"], a["dw"], a["db"]))
    dp.embedding_backward(a["dx"], a["ids"], a["table"].shape[0], scale=2.0, out=a["dtable"])


RESULTS = ("x", "y", "mean", "rstd", "loss", "stats", "dy", "loss2", "dy2", "dx", "dw", "db", "dtable")


@pytest.mark.parametrize("sizes", [dict(tokens=3, vocab=50, n=40001, k=70), dict(tokens=2100, vocab=3000, n=64, k=3)])
def test_captured_passes_of_other_shapes(sizes):
    """Rows shared by clusters of blocks, and a sort of several tiles, captured and replayed."""
    torch = pytest.importorskip("torch")
    import dpnp_b200 as dp

    tensors = _tensors(torch, 9, **sizes)
    torch.cuda.synchronize()
    _step(dp, _arrays(dp, tensors, dp.StreamQueue(0, stream=torch.cuda.current_stream().cuda_stream)))
    torch.cuda.synchronize()
    want = {k: tensors[k].clone() for k in RESULTS}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(dp, _views(dp, tensors, dp.StreamQueue(0, stream=torch.cuda.current_stream().cuda_stream)))
    for k in RESULTS:
        tensors[k].zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(tensors[k], want[k]) for k in RESULTS)


def _tensors(torch, seed, tokens=700, vocab=900, n=1031, k=5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    e = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    i = lambda hi, *s: torch.randint(0, hi, s, device="cuda", generator=gen, dtype=torch.int32)  # noqa: E731
    return dict(table=f(vocab, n), ids=i(vocab, tokens), w=f(n), b=f(n), t=f(tokens, k), idx=i(n, tokens, k), g=f(tokens),
                x=e(tokens, n), y=e(tokens, n), mean=e(tokens), rstd=e(tokens), loss=e(tokens), stats=e(tokens, 2),
                dy=e(tokens, n), loss2=e(tokens), dy2=e(tokens, n), dx=e(tokens, n), dw=e(n), db=e(n), dtable=e(vocab, n))


def _arrays(dp, tensors, queue):
    return {k: dp.from_dlpack(v, device=queue) for k, v in tensors.items()}


def _views(dp, tensors, queue):
    """The same without the exchange's synchronisation, which a capture does not allow."""
    return {k: dp.tensor.usm_ndarray._view(None, v.data_ptr(), tuple(v.shape), tuple(v.stride()),
                                           np.dtype(str(v.dtype).split(".")[1]), queue) for k, v in tensors.items()}


def test_two_captured_passes_replayed_side_by_side():
    """Passes captured into two graphs and replayed on two streams at once give the eager results."""
    torch = pytest.importorskip("torch")
    import dpnp_b200 as dp

    sets, want, graphs, streams = [], [], [], []
    for s in range(2):
        tensors = _tensors(torch, s)
        torch.cuda.synchronize()
        a = _arrays(dp, tensors, dp.StreamQueue(0, stream=torch.cuda.current_stream().cuda_stream))
        _step(dp, a)
        torch.cuda.synchronize()
        want.append({k: tensors[k].clone() for k in RESULTS})
        sets.append(tensors)
    for tensors in sets:
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            queue = dp.StreamQueue(0, stream=torch.cuda.current_stream().cuda_stream)
            _step(dp, _views(dp, tensors, queue))
        graphs.append(graph)
        streams.append(stream)
    for _ in range(3):
        for tensors in sets:
            for k in RESULTS:
                tensors[k].zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for tensors, w in zip(sets, want):
            for k in RESULTS:
                assert torch.equal(tensors[k], w[k]), k


def test_calls_on_two_queues_at_once():
    torch = pytest.importorskip("torch")
    import dpnp_b200 as dp

    sets = [_tensors(torch, s) for s in (4, 5)]
    torch.cuda.synchronize()
    queues = [dp.StreamQueue(0), dp.StreamQueue(0)]
    arrays = [_arrays(dp, t, q) for t, q in zip(sets, queues)]
    _step(dp, arrays[0])
    queues[0].wait()
    want = {k: sets[0][k].clone() for k in RESULTS}
    _step(dp, arrays[1])
    queues[1].wait()
    want1 = {k: sets[1][k].clone() for k in RESULTS}
    torch.cuda.synchronize()
    for _ in range(5):
        for a in arrays:
            _step(dp, a)
    for q in queues:
        q.wait()
    assert all(torch.equal(sets[0][k], want[k]) and torch.equal(sets[1][k], want1[k]) for k in RESULTS)


def test_writes_stay_inside_the_results():
    """With guard bytes around every block of the pool, odd sizes leave them intact."""
    import ctypes as C
    import gc

    import dpnp_b200 as dp
    from dpnp_b200 import _lib

    lib, check = _lib.lib, _lib.check

    def report():
        blocks, nbytes, first = C.c_int64(), C.c_int64(), (C.c_int64 * 3)()
        check(lib.dpb_debug_redzone_report(C.byref(blocks), C.byref(nbytes), first))
        return blocks.value, nbytes.value

    gc.collect()
    report()
    check(lib.dpb_set_tuning(b"redzones", 1))
    try:
        rng = np.random.default_rng(0)
        for dt in TYPES:
            for rows, n in ((1, 1), (3, 7), (33, 255), (5, 1025), (2, 20001), (1, 70001), (300, 31)):
                x, w, b, _ = norm_data(rows, n, dt, dt, n)
                y, m, r = dp.layer_norm(dev(x), dev(w), dev(b), return_stats=True)
                dp.layer_norm_backward(y, dev(x), m, r, dev(w))
                ids = rng.integers(-1, 50, rows).astype("i4")
                dp.embedding(dev(rng.normal(0, 1, (50, min(n, 2000))).astype(dt)), dev(ids))
                dp.embedding_backward(dev(x[:, :2000]), dev(ids), 50)
                z, t, idx, _ = distil_data(rows, n, 5, dt, n)
                dp.distillation_loss_and_grad(dev(z), dev(t), dev(idx))
                _, s = dp.distillation_loss(dev(z), dev(t), dev(idx), return_stats=True)
                dp.distillation_loss_backward(1.0, dev(z), dev(t), dev(idx), s)
        del y, m, r, s
        gc.collect()
        check(lib.dpb_device_synchronize())
        assert report() == (0, 0)
    finally:
        check(lib.dpb_set_tuning(b"redzones", 0))


# ------------------------------------------------------------- rows in two levels, more of them than groups of threads
def _two_levels(dp, kind, base):
    """An array (B, S, n) of rows in two levels, on the GPU and as NumPy sees it; `base` is (B, S + 3, n + 8)."""
    d, n, s = dev(base), base.shape[2] - 8, base.shape[1] - 3
    shape = (base.shape[0], s, n)
    if kind == "broadcast":                            # one matrix for all of the leading axis
        return dp.broadcast_to(d[0, :s, :n], shape), np.broadcast_to(base[0, :s, :n], shape)
    if kind == "broadcast, shifted":
        return dp.broadcast_to(d[0, 1:s + 1, 1:n + 1], shape), np.broadcast_to(base[0, 1:s + 1, 1:n + 1], shape)
    if kind == "broadcast inner":                      # one row for all of the inner axis
        return dp.broadcast_to(d[:, :1, :n], shape), np.broadcast_to(base[:, :1, :n], shape)
    return d[:, 2:s + 2, 8:], base[:, 2:s + 2, 8:]     # a slice: two different strides


TWO_LEVELS = ["broadcast", "broadcast, shifted", "broadcast inner", "slice"]
# (more rows than groups of threads that the GPU holds: a warp a row, then one to thirty-two warps a row)
MANY_ROWS = [(40, 130, 96), (43, 127, 37), (4, 330, 2048), (6, 301, 1001), (4, 90, 8192), (5, 70, 5001), (3, 20, 40000)]


@pytest.mark.parametrize("b,s,n", MANY_ROWS)
@pytest.mark.parametrize("kind", TWO_LEVELS)
@pytest.mark.parametrize("dt,wt", NORM_TYPES)
def test_layer_norm_of_rows_in_two_levels(dt, wt, kind, b, s, n):
    import dpnp_b200 as dp

    if dt == "f8" and n > 1000:
        b = max(2, b // 2)
    rng = np.random.default_rng(b * s + n)
    base = (rng.normal(0, 1, (b, s + 3, n + 8)) + rng.normal(0, 2, (b, s + 3, 1))).astype(dt)
    w, bias = (1 + 0.3 * rng.normal(0, 1, n)).astype(wt), (0.3 * rng.normal(0, 1, n)).astype(wt)
    d, x = _two_levels(dp, kind, base)
    dense = np.ascontiguousarray(x)
    y, mean, rstd = dp.layer_norm(d, dev(w), dev(bias), return_stats=True)
    check_norm(dense, w, bias, 1e-5, host(y), host(mean), host(rstd))
    big = dp.zeros(base.shape, dtype=dt)               # a result whose rows are in two levels
    dp.layer_norm(dev(dense), dev(w), dev(bias), out=big[:, 1:s + 1, 3:n + 3])
    got = host(big)
    check_norm(dense, w, bias, 1e-5, got[:, 1:s + 1, 3:n + 3], host(mean), host(rstd))
    got[:, 1:s + 1, 3:n + 3] = 0
    assert not got.any()


@pytest.mark.parametrize("b,s,n", MANY_ROWS)
@pytest.mark.parametrize("kind", TWO_LEVELS)
@pytest.mark.parametrize("dt,wt", NORM_TYPES)
def test_layer_norm_backward_of_rows_in_two_levels(dt, wt, kind, b, s, n):
    """x and dy in two levels, one after the other and both."""
    import dpnp_b200 as dp

    if dt == "f8" and n > 1000:
        b = max(2, b // 2)
    rng = np.random.default_rng(b * s + n)
    base = rng.normal(0, 1, (2, b, s + 3, n + 8)).astype(dt)
    w = (1 + 0.3 * rng.normal(0, 1, n)).astype(wt)
    (dx_, x), (dg, g) = (_two_levels(dp, kind, base[i]) for i in range(2))
    xc, gc = np.ascontiguousarray(x), np.ascontiguousarray(g)
    _, mean, rstd = dp.layer_norm(dev(xc), return_stats=True)
    m, r = host(mean), host(rstd)
    for dy, at in ((dg, dev(xc)), (dev(gc), dx_), (dg, dx_)):
        out = dp.layer_norm_backward(dy, at, mean, rstd, dev(w))
        check_norm_backward(xc, gc, w, m, r, *map(host, out))
    big = dp.zeros(base.shape[1:], dtype=dt)
    dp.layer_norm_backward(dg, dx_, mean, rstd, dev(w), out=(big[:, 1:s + 1, 3:n + 3], None, None))
    check_norm_backward(xc, gc, w, m, r, host(big)[:, 1:s + 1, 3:n + 3], None, None)


@pytest.mark.parametrize("kind", TWO_LEVELS)
@pytest.mark.parametrize("dt", TYPES)
def test_embedding_and_distillation_of_rows_in_two_levels(dt, kind):
    import dpnp_b200 as dp

    rng = np.random.default_rng(12)
    b, s, n = 30, 101, 75
    d, x = _two_levels(dp, kind, rng.normal(0, 2, (b, s + 3, n + 8)).astype(dt))
    x = np.ascontiguousarray(x)
    ids = rng.integers(-1, 60, (b, s)).astype("i4")
    check_embedding_backward(x, ids, 60, 0.5, host(dp.embedding_backward(d, dev(ids), 60, scale=0.5)), dt)
    t, idx = rng.normal(0, 2, (b, s, 4)).astype(ACC[dt]), rng.integers(-1, n, (b, s, 4)).astype("i4")
    loss, stats = dp.distillation_loss(d, dev(t), dev(idx), return_stats=True)
    check_distil(x, t, idx, 1.0, host(loss), None, host(stats))
    check_distil(x, t, idx, 1.0, None, host(dp.distillation_loss_backward(1.0, d, dev(t), dev(idx), stats)))
    loss, grad = dp.distillation_loss_and_grad(d, dev(t), dev(idx))
    check_distil(x, t, idx, 1.0, host(loss), host(grad))


@pytest.mark.parametrize("n", [1, 60, 64, 100, 256, 1000, 1024, 1537, 4100, 8192, 70001])
@pytest.mark.parametrize("dt", ["f4", "f8"])
def test_layer_norm_backward_of_constant_rows_of_large_values(dt, n):
    """x - mean is 0 there, and so is h, although mean * rstd is beyond the type's range: nothing of that product may
    come into the sums from threads that have no column."""
    import dpnp_b200 as dp

    rng = np.random.default_rng(n)
    rows, big = 9, 2.0**(123 if dt == "f4" else 1019)
    x = np.broadcast_to(big * (-1.0)**np.arange(rows)[:, None], (rows, n)).astype(dt)
    mean, rstd = np.ascontiguousarray(x[:, 0]), np.full(rows, 316.0, dt)
    assert 316.0 * big > float(np.finfo(dt).max)
    w, dy = (1 + 0.3 * rng.normal(0, 1, n)).astype(dt), rng.normal(0, 1, (rows, n)).astype(dt)
    for pad in (0, 1):                                 # rows on the 16-byte grid, and off it
        wide = np.zeros((2, rows, n + pad), dt)
        wide[0, :, pad:], wide[1, :, pad:] = dy, x
        out = dp.layer_norm_backward(dev(wide[0])[:, pad:], dev(wide[1])[:, pad:], dev(mean), dev(rstd), dev(w))
        check_norm_backward(x, dy, w, mean, rstd, *map(host, out))


def test_threads_with_rows_of_other_widths():
    """Two host threads at once in the C entry points, with widths for which one and the same kernel takes different
    amounts of shared memory: no call is refused, and the results are those of a single thread."""
    import ctypes as C
    import threading

    import dpnp_b200 as dp
    from dpnp_b200 import _lib

    def job(n, seed):
        q = dp.StreamQueue(0)
        x, w, b, rng = norm_data(5, n, "f4", "f4", seed)
        put = lambda a: dp.tensor.asarray(a, sycl_queue=q)  # noqa: E731
        a = dict(x=put(x), w=put(w), b=put(b), dy=put(rng.normal(0, 1, x.shape).astype("f4")),
                 **{k: put(np.zeros(x.shape, "f4")) for k in ("y", "dx")}, mean=put(np.zeros(5, "f4")), rstd=put(np.zeros(5, "f4")),
                 **{k: put(np.zeros(n, "f4")) for k in ("dw", "db")})
        keep = {k: v._descriptor() for k, v in a.items()}
        at = {k: C.byref(d[0]) for k, d in keep.items()}
        stream = C.c_void_p(q.stream)

        def step():
            return (_lib.lib.dpb_layer_norm(at["x"], at["w"], at["b"], 1e-5, at["y"], at["mean"], at["rstd"], stream),
                    _lib.lib.dpb_layer_norm_backward(at["dy"], at["x"], at["mean"], at["rstd"], at["w"], at["dx"], at["dw"],
                                                     at["db"], stream))

        def results():
            q.wait()
            return [dp.tensor.asnumpy(a[k]) for k in ("y", "mean", "rstd", "dx", "dw", "db")]

        return step, results, keep

    # forward: 64 KiB and 44 KiB; backward: 80 KiB and 55 KiB
    jobs = [job(8192, 1), job(5632, 2), job(4096, 3), job(2816, 4)]
    want = []
    for step, results, _ in jobs:
        assert step() == (_lib.OK, _lib.OK)
        want.append(results())
    refused, start = [], threading.Barrier(len(jobs))

    def loop(step):
        start.wait()
        for _ in range(3000):
            refused.extend(s for s in step() if s != _lib.OK)

    threads = [threading.Thread(target=loop, args=(step,)) for step, _, _ in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not refused
    for (_, results, _), w in zip(jobs, want):
        assert all(np.array_equal(p, q) for p, q in zip(results(), w))


@pytest.mark.parametrize("rows", [64, 512, 5000])
@pytest.mark.parametrize("dt", ["f4", "f8"])
def test_layer_norm_weight_gradients_add_their_parts_as_a_tree(dt, rows):
    """One large term and many of 1, of which each would be lost in a sum of its own with the large one.  The rows
    of a block are added one by one (at most rows / 64 + 1 of them here), the blocks' sums by 32 threads (at most
    rows / 2048 + 1 each), and those as a tree of 5 levels: that many roundings of the total, 2^24 or 2^53, each of them
    half a step of it at most, which is 1."""
    import dpnp_b200 as dp

    n = 1024
    dy = np.ones((rows, n), dt)
    dy[0] = 2.0**(24 if dt == "f4" else 53)
    if rows == 64:
        dy[32:] = 0
    total = float(np.sum(dy[1:, 0]))
    x, mean, rstd = np.ones((rows, n), dt), np.zeros(rows, dt), np.ones(rows, dt)
    _, dw, db = dp.layer_norm_backward(dev(dy), dev(x), dev(mean), dev(rstd))
    for g in (dw, db):
        more = host(g) - dy[0, 0]                      # exact: both are above 2^24 (2^53)
        assert np.all(np.abs(more - total) <= rows // 64 + 1 + rows // 2048 + 1 + 5), (more[0], total)


@pytest.mark.parametrize("temp", [0.1, 0.5, 0.7, 1.0, 2.0])
@pytest.mark.parametrize("dt", TYPES)
def test_distillation_at_columns_of_the_lowest_value(dt, temp):
    """A teacher's entry at a masked column: the loss is p T times the mask's depth, a number of the type, although the
    depth over T is not when T is below 1."""
    rng = np.random.default_rng(13)
    for rows, vocab, k in ((6, 40, 3), (4, 5001, 5), (3, 70000, 4)):
        z = rng.normal(0, 2, (rows, vocab)).astype(dt)
        z[:, ::7] = np.finfo(dt).min
        idx = 7 * np.stack([rng.choice(vocab // 7, k, replace=False) for _ in range(rows)]).astype("i4")
        idx[:, 1:] += 1                                 # the other entries are at columns that are not masked
        t = rng.normal(0, 1, (rows, k)).astype(ACC[dt])
        t[:, 0] -= 2 * temp
        loss, grad, _ = run_distil(z, t, idx, temp)
        if temp <= 1:                                   # p T < 1; its value is compared in run_distil
            assert np.isfinite(loss).all()


@pytest.mark.parametrize("dt,wt,widths", [("f4", "f4", (253, 257, 333, 381, 385, 401, 509, 513)), ("f8", "f8", (127, 129, 165, 191, 193, 255, 257)),
                                          ("f2", "f2", (505, 513, 737, 761, 769, 865, 1017, 1025)),
                                          ("f2", "f4", (505, 513, 737, 761, 769, 865, 1017, 1025))])
def test_layer_norm_of_shifted_rows_of_one_warp(dt, wt, widths):
    """Rows off the 16-byte grid on both sides of the lengths between which a warp takes a row by four accesses."""
    import dpnp_b200 as dp

    for n in widths:
        for rows in (1, 9, 3001):
            x, w, b, _ = norm_data(rows, n, dt, wt, n + rows)
            y, mean, rstd = dp.layer_norm(dev(x), dev(w), dev(b), return_stats=True)
            check_norm(x, w, b, 1e-5, host(y), host(mean), host(rstd))


FIRST_CALLS_CAPTURED = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import torch
import dpnp_b200 as dp
from test_gpu_row_operators import RESULTS, _arrays, _step, _tensors, _views

t = _tensors(torch, 3, tokens=40, vocab=50, n=8192, k=300)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    _step(dp, _views(dp, t, dp.StreamQueue(0, stream=torch.cuda.current_stream().cuda_stream)))
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
got = {{k: t[k].clone() for k in RESULTS}}
for k in RESULTS:
    t[k].zero_()
torch.cuda.synchronize()
_step(dp, _arrays(dp, t, dp.StreamQueue(0, stream=torch.cuda.current_stream().cuda_stream)))
torch.cuda.synchronize()
assert all(torch.equal(t[k], got[k]) for k in RESULTS)
"""


def test_first_calls_of_a_program_within_a_capture():
    """A program that captures its step without a pass before: what the library sets up once a device, the pool of
    the scratch and the kernels' shared memory, is set up during the capture."""
    import os
    import subprocess
    import sys

    pytest.importorskip("torch")
    tests = os.path.dirname(os.path.abspath(__file__))
    code = FIRST_CALLS_CAPTURED.format(root=os.path.dirname(tests), tests=tests)
    proc = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stderr[-3000:]
