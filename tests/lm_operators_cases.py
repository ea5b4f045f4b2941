"""The language-model operators against plain 64-bit statements of the same
mathematics: token embedding and its gradient, log probabilities with entropy
and alternatives and their gradient, the norm over many arrays and clipping.

The functions run twice: on a B200 (test_lm_operators_gpu.py) and, at the same
small sizes, on the CPU through the SIMT emulator behind a stand-in for the
CUDA driver (test_lm_operators_emulated.py). They take `api` and `ctx`.

Tolerances. u = 2^-24 is half a step of float, 2^-11 of half. A result rounded
once to half may be off by 2^-11 relative (2^-25 absolute near zero, half a
step of the smallest halfs) beyond what float arithmetic leaves.
"""
import numpy as np
import pytest

U = {np.dtype(np.float16): 2.0 ** -11, np.dtype(np.float32): 2.0 ** -24, np.dtype(np.float64): 2.0 ** -53}
TINY = {np.dtype(np.float16): 2.0 ** -25, np.dtype(np.float32): 2.0 ** -149, np.dtype(np.float64): 0.0}
INF = float("inf")


def put(api, ctx, a):
    return api.GpuArray.from_numpy(ctx, np.ascontiguousarray(a))


def strided(api, ctx, a, pad=3, fill=77):
    """`a` as a device view whose dimensions are all spaced out (every one but the last by a gap
    of `pad` entries), and the whole buffer, so that what lies between can be looked at."""
    shape = tuple(n + pad for n in a.shape)
    host = np.full(shape, fill, a.dtype)
    host[tuple(slice(1, 1 + n) for n in a.shape)] = a
    whole = api.GpuArray.from_numpy(ctx, host)
    return whole[tuple(slice(1, 1 + n) for n in a.shape)], whole, host


def spread(api, ctx, a):
    """`a` as a device view with every element two apart along the last axis."""
    host = np.repeat(a, 2, axis=-1)
    host[..., 1::2] = 0
    return api.GpuArray.from_numpy(ctx, host)[(slice(None),) * (a.ndim - 1) + (slice(0, 2 * a.shape[-1] - 1, 2),)]


def at_offset(api, ctx, a, k):
    """`a`, contiguous, starting k elements into its buffer and ending with it."""
    flat = np.zeros(a.size + k, a.dtype)
    flat[k:] = a.ravel()
    g = api.GpuArray.from_numpy(ctx, flat)[k:]
    return g.reshape(a.shape, nocopy=True)


def close(got, want, tol, what=""):
    """|got - want| <= tol elementwise; the same infinities and NaNs."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    odd = ~np.isfinite(want)
    assert (np.isnan(got) == np.isnan(want)).all(), what + ": NaNs differ"
    assert (got[odd & ~np.isnan(want)] == want[odd & ~np.isnan(want)]).all(), what + ": infinities differ"
    d = np.abs(got[~odd] - want[~odd])
    t = np.broadcast_to(np.asarray(tol, np.float64), want.shape)[~odd]
    assert (d <= t).all(), "%s: off by %g where %g is allowed" % (what, (d - t).max() + t[(d - t).argmax()], t[(d - t).argmax()])


# ------------------------------------------------------------------ embedding

def embed_formula(table, ids, scale, pad):
    out = table.astype(np.float64)[ids] * scale      # NumPy's negative indices are the rule
    if pad is not None:
        out[ids == pad] = 0
    return out


def embed_tol(want, dtype, f64):
    """one product in float (or double) and one rounding to the result's type"""
    u = U[np.dtype(np.float64)] if f64 else U[np.dtype(np.float32)]
    return np.abs(want) * 1.01 * (u + U[np.dtype(dtype)]) + TINY[np.dtype(dtype)]


EMBED_WIDTHS = [1, 2, 7, 8, 64, 100, 257, 1024]


@pytest.mark.parametrize("width", EMBED_WIDTHS)
@pytest.mark.parametrize("table_dtype,out_dtype", [("f2", "f2"), ("f4", "f4"), ("f2", "f4"), ("f4", "f2"), ("f8", "f8"), ("f2", "f8"), ("f8", "f2")])
def test_embed_types_and_widths(api, ctx, rng, width, table_dtype, out_dtype):
    table = rng.standard_normal((23, width)).astype(table_dtype)
    ids = rng.integers(-23, 23, 11).astype(np.int64)
    out = api.GpuArray.empty(ctx, (11, width), out_dtype)
    api.embed(out, put(api, ctx, table), put(api, ctx, ids), scale=0.75, check=True)
    want = embed_formula(table, ids, 0.75, None)
    close(out.to_numpy(), want, embed_tol(want, out_dtype, "f8" in (table_dtype, out_dtype)))


@pytest.mark.parametrize("width", [1, 8, 11])
def test_embed_and_gradient_round_doubles_to_halfs_once(api, ctx, width):
    """doubles next to the middle between two halfs: by way of float they would come to lie on it,
    and go to the even one"""
    step = 2.0 ** -10
    k = np.arange(23 * width).reshape(23, width)
    middle = (1 + step / 2 + step * (k % 1000)) * 2.0 ** (k % 9 - 4) * (-1.0) ** k
    v = middle * (1 + 2.0 ** -40 * (1 - 2 * (k // 2 % 2)))
    v[0, 0], v[1, 0], v[2, 0] = 2.0 ** -24 * (0.5 + 2.0 ** -40), 65520 * (1 - 2.0 ** -40), 1e300     # smallest, largest, infinite
    with np.errstate(over="ignore"):
        want = v.astype(np.float16)                        # one rounding to nearest
        assert (want != v.astype(np.float32).astype(np.float16)).any()
    ids = np.arange(23)[::-1].astype(np.int64)
    out = api.GpuArray.empty(ctx, (23, width), np.float16)
    api.embed(out, put(api, ctx, v), put(api, ctx, ids), check=True)
    assert (out.to_numpy() == want[ids]).all()
    op = api.GpuEmbedGrad(ctx)
    op(out, put(api, ctx, v), put(api, ctx, ids), check=True)
    assert (out.to_numpy() == want[ids]).all()
    # sorted tokens: six times the row more for the first three, in parts of 2^-6; a sum's few roundings
    # to double are far below its distance of 2^-40 to a middle
    many = np.concatenate([ids, np.repeat(ids[:3], 64 * 6)])
    up = np.concatenate([v, np.repeat(v[:3] / 64, 64 * 6, 0)])
    op(out, put(api, ctx, up), put(api, ctx, many), check=True)
    sums = v.copy()
    sums[:3] *= 7
    with np.errstate(over="ignore"):
        assert (out.to_numpy() == sums.astype(np.float16)[ids]).all()


@pytest.mark.parametrize("id_dtype", ["i4", "u4", "i8", "u8"])
@pytest.mark.parametrize("shape", [(), (1,), (5,), (2, 3), (2, 3, 2), (0,), (3, 0)])
def test_embed_ids_of_any_rank_and_type(api, ctx, rng, id_dtype, shape):
    table = rng.standard_normal((9, 12)).astype(np.float32)
    ids = rng.integers(0, 9, shape).astype(id_dtype)
    out = api.GpuArray.empty(ctx, shape + (12,), np.float32)
    api.embed(out, put(api, ctx, table), api.GpuArray.from_numpy(ctx, ids), pad=4)
    want = embed_formula(table, ids.astype(np.int64), 1.0, 4)
    assert (out.to_numpy() == want).all()              # scale 1: exact


@pytest.mark.parametrize("dtype", ["f2", "f4"])
def test_embed_strides_of_everything(api, ctx, rng, dtype):
    """a table with a row pitch, tokens[:, :-1] of a longer array, an out with gaps; then every
    element two apart: nothing between is touched"""
    table = rng.standard_normal((13, 24)).astype(dtype)
    tokens = rng.integers(0, 13, (3, 6)).astype(np.int32)
    t, _, _ = strided(api, ctx, table)
    ids = put(api, ctx, tokens)[:, :-1]
    out, whole, host = strided(api, ctx, np.zeros((3, 5, 24), dtype))
    api.embed(out, t, ids, scale=2.0, check=True)
    want = host.copy()
    want[1:4, 1:6, 1:25] = embed_formula(table, tokens[:, :-1], 2.0, None)
    assert (whole.to_numpy() == want).all()
    t2 = spread(api, ctx, table)
    back = put(api, ctx, tokens)[:, ::-1]              # negative stride
    out2 = api.GpuArray.empty(ctx, (24, 3, 6), dtype).transpose((1, 2, 0))
    api.embed(out2, t2, back, scale=2.0)
    assert (out2.to_numpy() == embed_formula(table, tokens[:, ::-1], 2.0, None)).all()


def test_embed_rows_out_of_range_are_reported_and_left(api, ctx, rng):
    table = rng.standard_normal((5, 40)).astype(np.float32)
    ids = np.array([0, 5, -5, -6, 2 ** 40, -2 ** 40, 4], np.int64)
    before = np.full((7, 40), 3.5, np.float32)
    out = put(api, ctx, before)
    api.embed(out, put(api, ctx, table), put(api, ctx, ids))       # not reported
    want = before.copy()
    for i, r in ((0, 0), (2, 0), (6, 4)):
        want[i] = table[r]
    assert (out.to_numpy() == want).all()
    with pytest.raises(api.GpuArrayException) as e:
        api.embed(out, put(api, ctx, table), put(api, ctx, ids), check=True)
    assert e.value.code == api.GA_VALUE_ERROR
    api.embed(out, put(api, ctx, table), put(api, ctx, ids), pad=5)   # again unreported
    want[1] = 0
    assert (out.to_numpy() == want).all()
    api.embed(api.GpuArray.empty(ctx, (1, 40), np.float32), put(api, ctx, table), put(api, ctx, ids[:1]), check=True)
    # an unsigned id of 2^64 - 1 is no negative one
    with pytest.raises(api.GpuArrayException):
        api.embed(api.GpuArray.empty(ctx, (1, 40), np.float32), put(api, ctx, table),
                  put(api, ctx, np.array([2 ** 64 - 1], np.uint64)), check=True)


def grad_formula(rows, dout, ids, scale, pad, base=None):
    width = dout.shape[-1]
    out = np.zeros((rows, width)) if base is None else base.astype(np.float64)
    size = np.zeros((rows, width)) if base is None else np.abs(base.astype(np.float64))
    flat, up = ids.reshape(-1), dout.reshape(-1, width).astype(np.float64)
    counts = np.zeros(rows)
    for t, i in enumerate(flat):
        if pad is not None and i == pad:
            continue
        if -rows <= i < rows:
            out[i] += scale * up[t]
            size[i] += abs(scale) * np.abs(up[t])
            counts[i] += 1
    return out, size, counts


def grad_tol(want, size, counts, dtype, f64):
    """n additions, a product and the sum with what was there, in float (or double): at most
    (n + 2) half steps of the sum of magnitudes; then one rounding to the result's type"""
    u = U[np.dtype(np.float64)] if f64 else U[np.dtype(np.float32)]
    return 1.01 * ((counts + 2)[:, None] * u * size + U[np.dtype(dtype)] * np.abs(want)) + TINY[np.dtype(dtype)]


GRAD_CASES = [  # tokens, rows, width
    (1, 1, 1), (1, 5, 8), (2, 1, 3), (7, 3, 16), (40, 6, 5), (64, 64, 24), (100, 2, 9), (257, 30, 12), (300, 1, 4),
    (512, 40, 33), (1024, 9, 6),
]
SORTED_CASES = [  # more tokens than one launch of the direct kernel takes; one to three passes, runs across many chunks
    (1025, 3, 4, "f2", "f2", True), (2600, 600, 9, "f4", "f4", True), (2600, 600, 24, "f2", "f4", False),
    (5000, 511, 3, "f4", "f4", False), (1100, 300000, 1, "f4", "f4", True), (17000, 900, 2, "f2", "f2", False),
    (1500, 2, 130, "f8", "f8", True), (4096, 90, 3, "f4", "f4", True), (4097, 90, 3, "f2", "f4", False), (33000, 700, 2, "f4", "f4", True),
]


@pytest.mark.parametrize("tokens,rows,width", GRAD_CASES)
@pytest.mark.parametrize("dout_dtype,out_dtype", [("f2", "f2"), ("f4", "f4"), ("f2", "f4"), ("f8", "f8")])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embed_gradient(api, ctx, rng, tokens, rows, width, dout_dtype, out_dtype, accumulate):
    embed_gradient_case(api, ctx, rng, tokens, rows, width, dout_dtype, out_dtype, accumulate)


@pytest.mark.parametrize("case", SORTED_CASES, ids=str)
def test_embed_gradient_of_sorted_tokens(api, ctx, rng, case):
    embed_gradient_case(api, ctx, rng, *case)


def embed_gradient_case(api, ctx, rng, tokens, rows, width, dout_dtype, out_dtype, accumulate):
    dout = rng.standard_normal((tokens, width)).astype(dout_dtype)
    ids = np.minimum(rng.geometric(0.3, tokens) - 1, rows - 1).astype(np.int32)   # few rows, often
    base = rng.standard_normal((rows, width)).astype(out_dtype)
    op = api.GpuEmbedGrad(ctx)
    results = []
    for _ in range(2):
        dt = put(api, ctx, base)
        op(dt, put(api, ctx, dout), put(api, ctx, ids), scale=1.5, accumulate=accumulate, check=True)
        results.append(dt.to_numpy())
    assert (results[0] == results[1]).all()            # the same bits every time
    want, size, counts = grad_formula(rows, dout, ids, 1.5, None, base if accumulate else None)
    close(results[0], want, grad_tol(want, size, counts, out_dtype, "f8" in (dout_dtype, out_dtype)))
    untouched = counts == 0
    assert (results[0][untouched] == (base if accumulate else 0 * base)[untouched]).all()


@pytest.mark.parametrize("shape", [(), (0,), (3, 0), (1,), (2, 5), (2, 2, 3)])
@pytest.mark.parametrize("id_dtype", ["i4", "u4", "i8", "u8"])
def test_embed_gradient_ranks_padding_and_bad_ids(api, ctx, rng, shape, id_dtype):
    rows, width = 6, 10
    dout = rng.standard_normal(shape + (width,)).astype(np.float32)
    ids = rng.integers(0, rows + 2, shape).astype(id_dtype)        # some outside the table
    op = api.GpuEmbedGrad(ctx)
    dt = put(api, ctx, np.full((rows, width), 9, np.float32))
    op(dt, api.GpuArray.from_numpy(ctx, dout), api.GpuArray.from_numpy(ctx, ids), pad=2)
    want, size, counts = grad_formula(rows, dout, ids.astype(np.int64), 1.0, 2)
    close(dt.to_numpy(), want, grad_tol(want, size, counts, "f4", False))
    if (ids >= rows).any():
        with pytest.raises(api.GpuArrayException) as e:
            op(dt, api.GpuArray.from_numpy(ctx, dout), api.GpuArray.from_numpy(ctx, ids), pad=2, check=True)
        assert e.value.code == api.GA_VALUE_ERROR


@pytest.mark.parametrize("tokens", [0, 5, 1500])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embed_gradient_of_an_empty_table(api, ctx, accumulate, tokens):
    """no rows to write: nothing happens, and every id is outside the table"""
    op = api.GpuEmbedGrad(ctx)
    dt, dout = api.GpuArray.empty(ctx, (0, 8), np.float32), api.GpuArray.empty(ctx, (tokens, 8), np.float32)
    ids = api.GpuArray.from_numpy(ctx, np.zeros(tokens, np.int64))
    op(dt, dout, ids, accumulate=accumulate)
    op(dt, dout, ids, accumulate=accumulate, pad=0, check=True)
    if tokens:
        with pytest.raises(api.GpuArrayException) as e:
            op(dt, dout, ids, accumulate=accumulate, check=True)
        assert e.value.code == api.GA_VALUE_ERROR
    else:
        op(dt, dout, ids, accumulate=accumulate, check=True)


def test_embed_gradient_negative_ids_and_all_padding(api, ctx, rng):
    dout = rng.standard_normal((6, 4)).astype(np.float32)
    ids = np.array([-1, 3, -4, 0, 3, -5], np.int64)
    op = api.GpuEmbedGrad(ctx)
    dt = api.GpuArray.empty(ctx, (4, 4), np.float32)
    op(dt, put(api, ctx, dout), put(api, ctx, ids))
    want = np.zeros((4, 4))
    want[3] = dout[[0, 1, 4]].astype(np.float64).sum(0)
    want[0] = dout[[2, 3]].astype(np.float64).sum(0)
    close(dt.to_numpy(), want, 4 * 2.0 ** -24 * np.abs(dout).sum(0) + 0 * want)
    op(dt, put(api, ctx, dout), put(api, ctx, np.full(6, -1, np.int64)), pad=-1)
    assert (dt.to_numpy() == 0).all()


def test_embed_gradient_strides_and_growing_calls(api, ctx, rng):
    """one operator for calls of growing and shrinking size; strided ids, dout and dtable"""
    op = api.GpuEmbedGrad(ctx)
    for tokens, rows, width, dtype in ((5, 4, 8, "f4"), (1300, 9, 24, "f2"), (300, 4, 8, "f4"), (3000, 600, 6, "f2")):
        dout = rng.standard_normal((2, tokens, width)).astype(dtype)
        tok = rng.integers(0, rows, (2, tokens + 1)).astype(np.int64)
        d, _, _ = strided(api, ctx, dout)
        dt, whole, host = strided(api, ctx, np.zeros((rows, width), dtype))
        op(dt, d, put(api, ctx, tok)[:, 1:], scale=0.5)
        want, size, counts = grad_formula(rows, dout, tok[:, 1:], 0.5, None)
        close(dt.to_numpy(), want, grad_tol(want, size, counts, dtype, False))
        edge = whole.to_numpy()
        edge[1:1 + rows, 1:1 + width] = host[1:1 + rows, 1:1 + width]
        assert (edge == host).all()                    # nothing around it was written
    dout = rng.standard_normal((12, 7)).astype(np.float32)
    ids = rng.integers(0, 3, 12).astype(np.int32)
    dt = api.GpuArray.empty(ctx, (7, 3), np.float32).transpose()
    op(dt, put(api, ctx, dout.T.copy()).transpose(), spread(api, ctx, ids))
    want, size, counts = grad_formula(3, dout, ids, 1.0, None)
    close(dt.to_numpy(), want, grad_tol(want, size, counts, "f4", False))


def test_embed_gradient_of_a_broadcast_upstream(api, ctx, rng):
    """one upstream row, and one upstream number, for all tokens (strides of 0); one id for all"""
    rows, width, tokens = 7, 8, 1200
    ids = rng.integers(0, rows, tokens).astype(np.int64)
    counts = np.bincount(ids, minlength=rows)
    row = put(api, ctx, rng.integers(-4, 4, width).astype(np.float32))
    op = api.GpuEmbedGrad(ctx)
    dt = api.GpuArray.empty(ctx, (rows, width), np.float32)
    for strides, each in (((0, 4), row.to_numpy()), ((0, 0), np.full(width, row.to_numpy()[0]))):
        up = api.GpuArray.from_pointer(ctx, row.devptr, (tokens, width), np.float32, strides=strides, nbytes=4 * width)
        op(dt, up, put(api, ctx, ids))
        assert (dt.to_numpy() == counts[:, None] * each).all()          # small whole numbers: exact
    one = put(api, ctx, ids[:1])
    every = api.GpuArray.from_pointer(ctx, one.devptr, (tokens,), np.int64, strides=(0,), nbytes=8)
    op(dt, up, every)
    want = np.zeros((rows, width))
    want[ids[0]] = tokens * row.to_numpy()[0]
    assert (dt.to_numpy() == want).all()


def test_embed_gradient_is_the_adjoint(api, ctx, rng):
    """<embed(E), D> = <E, grad(D)>, exactly in integers"""
    table = rng.integers(-8, 8, (15, 20)).astype(np.float32)
    ids = rng.integers(-15, 15, 60).astype(np.int64)
    d = rng.integers(-8, 8, (60, 20)).astype(np.float32)
    out = api.GpuArray.empty(ctx, (60, 20), np.float32)
    api.embed(out, put(api, ctx, table), put(api, ctx, ids), scale=0.5, pad=-3)
    dt = api.GpuArray.empty(ctx, (15, 20), np.float32)
    api.GpuEmbedGrad(ctx)(dt, put(api, ctx, d), put(api, ctx, ids), scale=0.5, pad=-3)
    assert (out.to_numpy().astype(np.float64) * d).sum() == (dt.to_numpy().astype(np.float64) * table).sum()


# ------------------------------------------------------------- log probabilities

def lp_formula(z, targets, scale, ignore=None):
    """logp, entropy, log p in 64 bits, with the conventions for rows without a distribution"""
    with np.errstate(all="ignore"):
        x = z.astype(np.float64) * scale
        m = x.max(-1, keepdims=True)
        empty = (m == -INF)[..., 0]
        e = np.exp(x - np.where(m == -INF, 0, m))
        s = e.sum(-1, keepdims=True)
        logs = x - np.where(m == -INF, 0, m) - np.log(s)
        p = e / s
        ent = -np.where(p > 0, p * np.where(p > 0, logs, 0), np.where(np.isnan(p), p, 0)).sum(-1)
    bad = np.isnan(s[..., 0])
    logs[logs < np.finfo(np.float32).min] = -INF        # results are floats: a scaled lowest value can lie below them
    logs[bad] = np.nan
    logs[empty] = -INF
    p[empty] = 0
    ent[empty] = 0
    logp = None
    if targets is not None:
        t = targets.astype(np.int64)
        ok = (t >= 0) & (t < z.shape[-1])
        logp = np.where(ok, np.take_along_axis(logs, np.where(ok, t, 0)[..., None], -1)[..., 0], np.nan)
        if ignore is not None:
            logp[t == ignore] = 0
    return logp, ent, logs, p, empty


def lp_tols(z, scale, p):
    """Errors of one pass in float. A term e^y: y = (z - m) scale log2(e) has three roundings, each
    half a step of |y|, and the scale's log2(e) one: 4 u |y| in the exponent; the instruction for
    2^y is within 2^-22 relative. Terms are added in a tree over threads whose longest chain is n
    terms: (n + 12) u; rescalings (at most one per 32 or 4 terms, each 2^-22 and two products) are
    counted as 2^-21 for each of the up to 20 that change a sum noticeably. The sum's relative
    error r is its logarithm's absolute one; the logarithm adds 2 u of its size."""
    V = z.shape[-1]
    with np.errstate(all="ignore"):
        zz = np.where(np.isfinite(z), z, np.nan).astype(np.float64) * scale
        d = np.nan_to_num(np.nanmax(np.where(np.isnan(zz), -INF, zz), -1, keepdims=True) - zz, nan=0.0, posinf=0.0)
    ydp = (np.abs(d) * p).sum(-1)                       # mean |x - m| under p
    chain = min(V, 64 + V // 64)
    u = 2.0 ** -24
    r = 4 * u * ydp + 2.0 ** -22 + (chain + 12) * u + 20 * 2.0 ** -21
    lns = np.log(V) + 1
    return r + 2 * u * lns, (r * (2 + ydp + lns) + 4 * u * (lns + ydp)), d


def rows_of_logits(rng, rows, V, dtype, kind):
    z = (rng.standard_normal((rows, V)) * 2).astype(np.float32)
    z[:, rng.integers(0, V, 1 + V // 50)] += 6
    if kind == "masked":
        z[rng.random((rows, V)) < 0.4] = -INF
        z[rows // 2] = -INF
        if rows > 2:
            z[0] = -INF
            z[0, V // 2] = 1.5                          # one entry is left
    if kind == "lowest":
        z[rng.random((rows, V)) < 0.4] = np.finfo(dtype).min
        z[rows // 2] = np.finfo(dtype).min              # uniform over everything
        if rows > 2:
            z[0] = -INF
            z[0, -1] = np.finfo(dtype).min              # all the mass on one lowest value
    if kind == "ties":
        z = np.round(z)
        z[-1] = 2.5
    if kind == "large":
        z *= 300
    return z.astype(dtype)


def check_top(api, z, k, values, ids, logs, tol, empty):
    """the largest logits, equal ones by the lower index, NaNs last"""
    with np.errstate(invalid="ignore"):
        keyed = np.where(np.isnan(z), -INF, z.astype(np.float64))
    for r in range(z.shape[0]):
        order = np.lexsort((np.arange(z.shape[1]), np.isnan(z[r]), -keyed[r]))
        order = np.concatenate([order[~np.isnan(z[r][order])], order[np.isnan(z[r][order])]])[:k]
        assert (ids[r] == order).all(), (r, ids[r], order)
        close(values[r], logs[r][order], tol[r], "row %d" % r)


SHAPES = [(1, 1), (3, 2), (4, 7), (5, 33), (3, 256), (3, 1000), (40, 150), (34, 1111), (2, 2049), (2, 4500), (1, 9001)]


@pytest.mark.parametrize("dtype", ["f2", "f4"])
@pytest.mark.parametrize("kind", ["plain", "masked", "lowest", "ties", "large"])
@pytest.mark.parametrize("rows,V", SHAPES)
def test_logprobs(api, ctx, rng, dtype, kind, rows, V):
    top = min(V, [0, 1, 5, 20, 32, 32][(rows + V) % 6])
    z = rows_of_logits(rng, rows, V, dtype, kind)
    targets = rng.integers(0, V, rows).astype(np.int64)
    scale = [1.0, 0.7, 1.3, 100.0][V % 4]
    op = api.GpuLogProbs(ctx, dtype, np.int64, top=top)
    lead = (rows,)
    d = {n: api.GpuArray.empty(ctx, s, t) for n, s, t in (
        ("logp", lead, np.float32), ("entropy", lead, np.float32), ("stats", lead + (2,), np.float32))}
    if top:
        d["top_logp"] = api.GpuArray.empty(ctx, lead + (top,), np.float32)
        d["top_ids"] = api.GpuArray.empty(ctx, lead + (top,), np.int64)
    op(put(api, ctx, z), put(api, ctx, targets), scale=scale, check=True, **d)
    logp, ent, logs, p, empty = lp_formula(z, targets, scale)
    tol_lse, tol_ent, gap = lp_tols(z, scale, p)
    with np.errstate(invalid="ignore"):
        t_gap = np.take_along_axis(gap, targets[:, None], -1)[:, 0]
        close(d["logp"].to_numpy(), logp, tol_lse + 4 * 2.0 ** -24 * (t_gap + np.log(V)), "logp")
    close(d["entropy"].to_numpy(), ent, tol_ent, "entropy")
    st = d["stats"].to_numpy().astype(np.float64)
    assert (st[:, 0] == z.astype(np.float64).max(-1)).all()
    with np.errstate(all="ignore"):
        s = np.exp((z.astype(np.float64) - np.where(empty, 0, z.max(-1))[:, None]) * scale).sum(-1)
        close(st[:, 1], np.log(s), tol_lse, "log of the sum")
    if top:
        ids = d["top_ids"].to_numpy()
        with np.errstate(invalid="ignore"):
            g = np.take_along_axis(gap, ids, -1)
        check_top(api, z, top, d["top_logp"].to_numpy(), ids, logs, tol_lse[:, None] + 4 * 2.0 ** -24 * (g + np.log(V)), empty)


@pytest.mark.parametrize("dtype", ["f2", "f4"])
@pytest.mark.parametrize("kind", ["plain", "masked", "ties"])
@pytest.mark.parametrize("V", [2, 61, 250])
def test_logprobs_of_short_rows_within_their_few_roundings(api, ctx, rng, dtype, kind, V):
    """Rows of at most 64 vectors: a lane has three of them at most. A term e^y has 4 u |y| and the
    instruction's 4 u as in lp_tols, along with what rescaling adds to its exponent; a lane adds at most
    13 numbers, five additions join the lanes; two rescalings in a lane, that of the lanes' join and the
    one that takes back a folded product have 6 u each: 46 u. The logarithm is off by 2 u of its size,
    the difference to the target by 3 u of its own, the result by u."""
    u = 2.0 ** -24
    z = rows_of_logits(rng, 37, V, dtype, kind)
    targets = rng.integers(0, V, 37).astype(np.int64)
    lp, st = api.GpuArray.empty(ctx, (37,), "f4"), api.GpuArray.empty(ctx, (37, 2), "f4")
    op = api.GpuLogProbs(ctx, dtype, np.int64)
    for g in (put(api, ctx, z), at_offset(api, ctx, z, 1)):
        op(g, put(api, ctx, targets), logp=lp, stats=st, scale=1.0)
        want, _, _, p, empty = lp_formula(z, targets, 1.0)
        gap = lp_tols(z, 1.0, p)[2]
        with np.errstate(invalid="ignore", divide="ignore"):
            ls = np.log(np.exp(z.astype(np.float64) - np.where(empty, 0, z.max(-1).astype(np.float64))[:, None]).sum(-1))
        tol = 1.01 * u * (4 * (gap * p).sum(-1) + 46 + 2 * np.where(empty, 0, ls))
        close(st.to_numpy()[:, 1], np.where(empty, -INF, ls), tol, "log of the sum")
        t_gap = np.take_along_axis(gap, targets[:, None], -1)[:, 0]
        close(lp.to_numpy(), want, tol + 1.01 * u * (3 * t_gap + np.where(np.isfinite(want), np.abs(want), 0)), "logp")


@pytest.mark.parametrize("dtype", ["f2", "f4"])
def test_logprobs_rows_that_hide_their_largest_in_few_threads(api, ctx, rng, dtype):
    """values that rise with period 2048 (or 1024) vectors put the largest in the same threads; a
    row of one value; a row of NaNs and infinities"""
    V, k = 40001, 32
    per = 256 * (8 if dtype == "f2" else 4)
    z = np.zeros((4, V), np.float32)
    i = np.arange(V)
    z[0] = np.where(i % per < 8, 10 + (i // per) * 0.25 + (i % per) * 0.03125, -5)
    z[1] = 3.0
    z[2] = rng.standard_normal(V)
    z[2, ::3] = np.nan
    z[2, 1::3] = -INF
    z[3] = rng.standard_normal(V)
    z[3, [7, 39000]] = INF
    z = z.astype(dtype)
    op = api.GpuLogProbs(ctx, dtype, np.int32, top=k)
    logp, ent = (api.GpuArray.empty(ctx, (4,), np.float32) for _ in range(2))
    tv, ti = api.GpuArray.empty(ctx, (4, k), np.float32), api.GpuArray.empty(ctx, (4, k), np.int32)
    targets = np.array([5, 6, 8, 7], np.int32)
    op(put(api, ctx, z), put(api, ctx, targets), logp=logp, entropy=ent, top_logp=tv, top_ids=ti)
    want, went, logs, p, empty = lp_formula(z, targets, 1.0)
    assert np.isnan(want[2:]).all() and np.isnan(logp.to_numpy()[2:]).all() and np.isnan(ent.to_numpy()[2:]).all()
    ids = ti.to_numpy()
    for r in range(4):
        v = z[r].astype(np.float64)
        order = np.concatenate([np.lexsort((i, -np.nan_to_num(v, nan=-INF, posinf=INF, neginf=-INF)))])
        order = np.concatenate([order[~np.isnan(v[order])], order[np.isnan(v[order])]])[:k]
        assert (ids[r] == order).all(), r
    assert np.isnan(tv.to_numpy()[2:]).all()
    tol = lp_tols(z[:2], 1.0, p[:2])[0]
    close(tv.to_numpy()[:2], np.take_along_axis(logs[:2], ids[:2].astype(np.int64), -1), tol[:, None] + 1e-5)


@pytest.mark.parametrize("dtype", ["f2", "f4"])
@pytest.mark.parametrize("V", [5, 50, 1001, 2600])
def test_logprobs_strides_and_alignments(api, ctx, rng, dtype, V):
    """rows that start anywhere, spaced logits, tokens[:, 1:], destinations with gaps, three
    leading dimensions"""
    z = rows_of_logits(rng, 12, V, dtype, "plain").reshape(2, 3, 2, V)
    targets = rng.integers(0, V, (2, 3, 2)).astype(np.int32)
    logp, ent, logs, p, _ = lp_formula(z, targets, 1.0)
    tl, te, gap = lp_tols(z, 1.0, p)
    tl = tl + 4 * 2.0 ** -24 * (np.take_along_axis(gap, targets[..., None].astype(np.int64), -1)[..., 0] + np.log(V))
    op = api.GpuLogProbs(ctx, dtype, np.int32, top=3)
    views = [strided(api, ctx, z, pad=1)[0], strided(api, ctx, z, pad=2)[0], spread(api, ctx, z),
             put(api, ctx, np.moveaxis(z, -1, 0)).transpose((1, 2, 3, 0))] + [at_offset(api, ctx, z, k) for k in (1, 3, 7)]
    for v in views:
        t = strided(api, ctx, targets)[0]
        lp, wl, hl = strided(api, ctx, np.zeros((2, 3, 2), np.float32))
        en, we, he = strided(api, ctx, np.zeros((2, 3, 2), np.float32))
        tv, wv, hv = strided(api, ctx, np.zeros((2, 3, 2, 3), np.float32))
        ti, wi, hi = strided(api, ctx, np.zeros((2, 3, 2, 3), np.int32))
        op(v, t, logp=lp, entropy=en, top_logp=tv, top_ids=ti, check=True)
        close(lp.to_numpy(), logp, tl)
        close(en.to_numpy(), ent, te)
        want = np.argsort(-z.astype(np.float64), -1, kind="stable")[..., :3]
        assert (ti.to_numpy() == want).all()
        close(tv.to_numpy(), np.take_along_axis(logs, want, -1), tl.max() + 1e-6)
        for w, h in ((wl, hl), (we, he), (wv, hv), (wi, hi)):
            edge, inner = w.to_numpy(), tuple(slice(1, n - 2) for n in h.shape)
            edge[inner] = h[inner]
            assert (edge == h).all()


def test_logprobs_ignored_and_bad_targets(api, ctx, rng):
    z = rows_of_logits(rng, 6, 70, "f4", "plain")
    z[1] = np.nan
    targets = np.array([3, -100, 70, -1, 69, -100], np.int64)
    op = api.GpuLogProbs(ctx, "f4", np.int64)
    logp = api.GpuArray.empty(ctx, (6,), np.float32)
    stats = api.GpuArray.empty(ctx, (6, 2), np.float32)
    gz, gt = put(api, ctx, z), put(api, ctx, targets)
    op(gz, gt, logp=logp, stats=stats, ignore=-100)
    got = logp.to_numpy()
    assert (got[[1, 5]] == 0).all() and np.isnan(got[[2, 3]]).all() and np.isfinite(got[[0, 4]]).all()
    dl = put(api, ctx, np.ones(6, np.float32))
    dz = put(api, ctx, np.full((6, 70), 5, np.float32))
    op.grad(dz, gz, gt, stats, dl, ignore=-100)
    g = dz.to_numpy()
    assert (g[[1, 5]] == 0).all() and np.isnan(g[[2, 3]]).all() and np.isfinite(g[[0, 4]]).all()
    for call in (lambda: op(gz, gt, logp=logp, ignore=-100, check=True), lambda: op.grad(dz, gz, gt, stats, dl, ignore=-100, check=True)):
        with pytest.raises(api.GpuArrayException) as e:
            call()
        assert e.value.code == api.GA_VALUE_ERROR
    op(put(api, ctx, z[:1]), put(api, ctx, targets[:1]), logp=api.GpuArray.empty(ctx, (1,), np.float32), check=True)


@pytest.mark.parametrize("dtype", ["f2", "f4"])
def test_logprobs_scales_near_the_largest_float(api, ctx, dtype):
    """refused where scale log2(e) is no float, and right below that"""
    V = api.GA_VALUE_ERROR
    z, t = put(api, ctx, np.array([[1, 1, 0.5, 1], [0, -0.25, -1, -2]], dtype)), put(api, ctx, np.array([1, 0], np.int64))
    e = api.GpuArray.empty
    op, lp, en, st = api.GpuLogProbs(ctx, dtype, np.int64), e(ctx, (2,), "f4"), e(ctx, (2,), "f4"), e(ctx, (2, 2), "f4")
    largest = float(np.finfo(np.float32).max) / np.log2(np.e)
    for bad in (largest * 1.0001, 2.4e38, 3e38, 3.4028235e38):
        refused(api, V, lambda: op(z, t, logp=lp, entropy=en, stats=st, scale=bad))
        refused(api, V, lambda: op.grad(z, z, t, st, lp, scale=bad))
    op(z, t, logp=lp, entropy=en, stats=st, scale=largest * 0.9999, check=True)
    # equal logits share the mass, the others have none; two roundings of a logarithm and its part
    close(lp.to_numpy(), [-np.log(3), 0], 8 * 2.0 ** -24)
    close(en.to_numpy(), [np.log(3), 0], 8 * 2.0 ** -24)
    dz = put(api, ctx, np.full((2, 4), 7, np.float32))
    op.grad(dz, z, t, st, put(api, ctx, np.full(2, 1e-38, np.float32)), scale=largest * 0.9999)
    a = np.float32(1e-38).astype(np.float64) * largest * 0.9999
    close(dz.to_numpy(), [[-a / 3, a * 2 / 3, 0, -a / 3], [0, 0, 0, 0]], 16 * 2.0 ** -24 * a)


@pytest.mark.parametrize("dtype", ["f2", "f4"])
@pytest.mark.parametrize("V", [1, 40, 5000])
def test_logprobs_stats_of_rows_with_nans_and_infinities(api, ctx, rng, dtype, V):
    """both numbers are NaN, and -inf in a row of -inf; the others are what they are alone"""
    z = rows_of_logits(rng, 6, V, dtype, "plain")
    z[0, V // 2] = np.nan
    z[1, V - 1] = INF
    z[2] = np.nan
    z[3, ::2] = INF
    z[4] = -INF
    st, one = api.GpuArray.empty(ctx, (6, 2), np.float32), api.GpuArray.empty(ctx, (1, 2), np.float32)
    op = api.GpuLogProbs(ctx, dtype, np.int32)
    op(put(api, ctx, z), stats=st)
    op(put(api, ctx, z[5:]), stats=one)
    got = st.to_numpy()
    assert np.isnan(got[:4]).all(), got
    assert (got[4] == -INF).all()
    assert got[5, 0] == one.to_numpy()[0, 0] == z[5].max() and abs(got[5, 1] - one.to_numpy()[0, 1]) <= 2 * lp_tols(z[5:], 1.0, lp_formula(z[5:], None, 1.0)[3])[0]


@pytest.mark.parametrize("dtype", ["f2", "f4"])
def test_logprobs_of_one_row_and_of_repeated_rows(api, ctx, rng, dtype):
    """a 1-d array of logits with 0-d results; the same row for every target (a stride of 0)"""
    V = 300
    z = rows_of_logits(rng, 1, V, dtype, "plain")
    op = api.GpuLogProbs(ctx, dtype, np.int64, top=2)
    e = api.GpuArray.empty
    gz = put(api, ctx, z[0])
    lp, tv, ti, st = e(ctx, (), "f4"), e(ctx, (2,), "f4"), e(ctx, (2,), "i8"), e(ctx, (2,), "f4")
    op(gz, api.GpuArray.from_numpy(ctx, np.array(7, np.int64)), logp=lp, top_logp=tv, top_ids=ti, stats=st, check=True)
    want, _, logs, p, _ = lp_formula(z, np.array([7]), 1.0)
    tol = lp_tols(z, 1.0, p)[0] + 1e-5
    close(lp.to_numpy(), want[0], tol[0])
    assert (ti.to_numpy() == np.argsort(-z[0].astype(np.float64), kind="stable")[:2]).all()
    dz = e(ctx, (V,), dtype)
    op.grad(dz, gz, api.GpuArray.from_numpy(ctx, np.array(7, np.int64)), st, api.GpuArray.from_numpy(ctx, np.array(2, np.float32)))
    g, p, logs, h = lp_grad_formula(z, np.array([7]), 1.0, np.array([2.0]), None)
    t = lp_grad_tol(z, 1.0, p, logs, h, np.array([2.0]), None, dtype)
    close(dz.to_numpy(), g[0], (t + U[np.dtype(dtype)] * (np.abs(g) + t) + TINY[np.dtype(dtype)])[0])
    many = api.GpuArray.from_pointer(ctx, gz.devptr, (50, V), dtype, strides=(0, gz.dtype.itemsize), nbytes=V * gz.dtype.itemsize)
    targets = rng.integers(0, V, 50)
    out = e(ctx, (50,), "f4")
    op(many, put(api, ctx, targets.astype(np.int64)), logp=out)
    close(out.to_numpy(), lp_formula(np.repeat(z, 50, 0), targets, 1.0)[0], tol)


def lp_grad_formula(z, targets, scale, a, b, ignore=None):
    logp, ent, logs, p, empty = lp_formula(z, targets, scale, ignore)
    t = targets.astype(np.int64)
    kept = np.ones(t.shape, bool) if ignore is None else t != ignore
    a = np.where(kept, a, 0.0)
    hot = np.zeros(z.shape)
    np.put_along_axis(hot, np.where(kept, t, 0)[..., None], 1.0, -1)
    g = a[..., None] * (hot - p)
    if b is not None:
        g = g - b[..., None] * p * (np.where(p > 0, logs, 0) + ent[..., None])
    g[empty] = 0
    return scale * g, p, logs, ent


def lp_grad_tol(z, scale, p, logs, ent, a, b, dtype):
    """p has the relative error of e^y, y = log2 p: 4 u |y| + 2^-22, and of the forward pass's log
    of the sum; the bracket a + b (log p + H) has 6 u of its parts' magnitudes and b times the
    error of H; three products, one sum at the target, one rounding."""
    tl, te, _ = lp_tols(z, scale, p)
    u = 2.0 ** -24
    with np.errstate(all="ignore"):
        l = np.where(p > 0, np.abs(logs), 0)
    rel = 4 * u * l + 2.0 ** -22 + tl[..., None] + 8 * u
    mag = np.abs(a)[..., None] + 0 * p
    extra = 0
    if b is not None:
        mag = mag + np.abs(b)[..., None] * (l + np.abs(ent)[..., None])
        extra = np.abs(b)[..., None] * te[..., None]
    want = p * mag * (rel + 6 * u) + p * extra + 2 * u * np.abs(a)[..., None]
    return 1.01 * scale * want


@pytest.mark.parametrize("dtype,out_dtype", [("f2", "f2"), ("f4", "f4"), ("f2", "f4")])
@pytest.mark.parametrize("kind", ["plain", "masked", "lowest", "large"])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (5, 33), (4, 256), (3, 1003), (2, 4500)])
@pytest.mark.parametrize("with_entropy", [False, True])
def test_logprobs_gradient(api, ctx, rng, dtype, out_dtype, kind, rows, V, with_entropy):
    z = rows_of_logits(rng, rows, V, dtype, kind)
    targets = rng.integers(0, V, rows).astype(np.int32)
    if rows > 3:
        targets[1] = -1
    scale = [1.0, 0.7][V % 2]
    a = rng.standard_normal(rows).astype(np.float32)
    b = rng.standard_normal(rows).astype(np.float32) if with_entropy else None
    op = api.GpuLogProbs(ctx, dtype, np.int32)
    gz, gt = put(api, ctx, z), put(api, ctx, targets)
    logp, ent = (api.GpuArray.empty(ctx, (rows,), np.float32) for _ in range(2))
    stats = api.GpuArray.empty(ctx, (rows, 2), np.float32)
    op(gz, gt, logp=logp, entropy=ent, stats=stats, scale=scale, ignore=-1)
    dz = put(api, ctx, np.full((rows, V), 7, out_dtype))
    more = dict(entropy=ent, dentropy=put(api, ctx, b)) if with_entropy else {}
    op.grad(dz, gz, gt, stats, put(api, ctx, a), scale=scale, ignore=-1, **more)
    want, p, logs, h = lp_grad_formula(z, targets, scale, a.astype(np.float64), None if b is None else b.astype(np.float64), -1)
    tol = lp_grad_tol(z, scale, p, logs, h, a, b, out_dtype)
    close(dz.to_numpy(), want, tol + U[np.dtype(out_dtype)] * (np.abs(want) + tol) + TINY[np.dtype(out_dtype)])
    if dtype == out_dtype:                              # in place
        op.grad(gz, gz, gt, stats, put(api, ctx, a), scale=scale, ignore=-1, **more)
        assert (gz.to_numpy() == dz.to_numpy()).all()


@pytest.mark.parametrize("dtype", ["f2", "f4"])
def test_logprobs_gradient_of_rows_with_nans_and_infinities(api, ctx, rng, dtype):
    """NaN throughout, but 0 in an ignored row whatever it holds"""
    z = rows_of_logits(rng, 5, 40, dtype, "plain")
    z[0, 3] = np.nan
    z[1, 4] = INF
    z[2] = np.nan
    z[3, ::2] = INF
    targets = np.array([1, 4, -1, -1, 6], np.int32)
    op = api.GpuLogProbs(ctx, dtype, np.int32)
    gz, gt = put(api, ctx, z), put(api, ctx, targets)
    lp, stats = api.GpuArray.empty(ctx, (5,), np.float32), api.GpuArray.empty(ctx, (5, 2), np.float32)
    op(gz, gt, logp=lp, stats=stats, ignore=-1)
    op.grad(gz, gz, gt, stats, put(api, ctx, np.ones(5, np.float32)), ignore=-1)
    g = gz.to_numpy()
    assert np.isnan(g[:2]).all() and (g[2:4] == 0).all() and np.isfinite(g[4]).all()


@pytest.mark.parametrize("dtype", ["f2", "f4"])
@pytest.mark.parametrize("with_entropy", [False, True])
def test_logprobs_gradient_of_bad_targets_in_empty_rows(api, ctx, dtype, with_entropy):
    """a target outside the vocabulary gives a logp and a gradient row of NaN, in a row without a
    logit above -inf too; 0 there for any other target"""
    V = 70
    z = np.full((5, V), -INF, dtype)
    z[4] = 0.5
    t = np.array([V, -1, 3, -7, 1000], np.int64)         # outside, ignored, inside, outside, outside
    op = api.GpuLogProbs(ctx, dtype, np.int64)
    gz, gt = put(api, ctx, z), put(api, ctx, t)
    e = api.GpuArray.empty
    lp, en, st = e(ctx, (5,), "f4"), e(ctx, (5,), "f4"), e(ctx, (5, 2), "f4")
    op(gz, gt, logp=lp, entropy=en, stats=st, ignore=-1)
    assert (np.isnan(lp.to_numpy()) == [True, False, False, True, True]).all()
    dz, one = put(api, ctx, np.full((5, V), 7, dtype)), put(api, ctx, np.ones(5, np.float32))
    op.grad(dz, gz, gt, st, one, ignore=-1, **(dict(entropy=en, dentropy=one) if with_entropy else {}))
    got = dz.to_numpy()
    assert np.isnan(got[[0, 3, 4]]).all() and (got[1:3] == 0).all()


@pytest.mark.parametrize("dtype", ["f2", "f4"])
def test_logprobs_gradient_strides_and_broadcast_inputs(api, ctx, rng, dtype):
    V = 53
    z = rows_of_logits(rng, 6, V, dtype, "plain").reshape(2, 3, V)
    targets = rng.integers(0, V, (2, 3)).astype(np.int64)
    a = np.full((2, 3), -0.25)
    want, p, logs, h = lp_grad_formula(z, targets, 1.0, a, None)
    tol = lp_grad_tol(z, 1.0, p, logs, h, a, None, dtype)
    tol = tol + U[np.dtype(dtype)] * (np.abs(want) + tol) + TINY[np.dtype(dtype)]
    op = api.GpuLogProbs(ctx, dtype, np.int64)
    one = put(api, ctx, np.array([-0.25], np.float32))
    for v in (strided(api, ctx, z, pad=1)[0], spread(api, ctx, z), at_offset(api, ctx, z, 5)):
        stats = strided(api, ctx, np.zeros((2, 3, 2), np.float32))[0]
        t = put(api, ctx, np.concatenate([targets, targets], 1))[:, 3:]
        lp = api.GpuArray.empty(ctx, (2, 3), np.float32)
        op(v, t, logp=lp, stats=stats)
        every = api.GpuArray.from_pointer(ctx, one.devptr, (2, 3), np.float32, strides=(0, 0), nbytes=4)
        for dz, whole, host in (strided(api, ctx, np.zeros(z.shape, dtype), pad=2), strided(api, ctx, np.zeros(z.shape, dtype), pad=1)):
            op.grad(dz, v, t, stats, every)
            close(dz.to_numpy(), want, tol)
            edge, inner = whole.to_numpy(), tuple(slice(1, 1 + n) for n in z.shape)
            edge[inner] = host[inner]
            assert (edge == host).all()
        far = api.GpuArray.empty(ctx, (V, 2, 3), dtype).transpose((1, 2, 0))
        op.grad(far, v, t, stats, every)
        close(far.to_numpy(), want, tol)


def test_logprobs_gradient_agrees_with_differences(api, ctx, rng):
    """central differences of sum(a logp + b entropy), taken from the kernel's own float results:
    a step of 1/16 leaves a truncation error of h^2 / 6 times a third derivative below 4 (softmax
    derivatives of order three are at most 1 for logp, times |log p| for the entropy, |a|, |b| <= 1,
    |log p| < 4: 2^-8 / 6 * 5 < 0.0033), and rounding of 2 * 8 results of at most 8 u * 8 over 2 h:
    below 0.0002"""
    rows, V, step = 4, 6, 0.0625
    z = np.round(rng.uniform(-1, 1, (rows, V)) * 64).astype(np.float32) / 64
    t = rng.integers(0, V, rows).astype(np.int32)
    a, b = rng.uniform(-1, 1, rows).astype(np.float32), rng.uniform(-1, 1, rows).astype(np.float32)
    op = api.GpuLogProbs(ctx, "f4", np.int32)
    logp, ent = (api.GpuArray.empty(ctx, (rows,), np.float32) for _ in range(2))
    stats, dz = api.GpuArray.empty(ctx, (rows, 2), np.float32), api.GpuArray.empty(ctx, (rows, V), np.float32)
    gt = put(api, ctx, t)

    def value(x):
        op(put(api, ctx, x), gt, logp=logp, entropy=ent, stats=stats)
        return a.astype(np.float64) * logp.to_numpy() + b.astype(np.float64) * ent.to_numpy()
    value(z)
    op.grad(dz, put(api, ctx, z), gt, stats, put(api, ctx, a), entropy=ent, dentropy=put(api, ctx, b))
    got = dz.to_numpy()
    for j in range(V):
        hi, lo = z.copy(), z.copy()
        hi[:, j] += step
        lo[:, j] -= step
        assert np.abs((value(hi) - value(lo)) / (2 * step) - got[:, j]).max() <= 0.0035


# --------------------------------------------------------------- norm and clipping

def clip_formula(arrays, scale, limit):
    with np.errstate(all="ignore"):
        norm = abs(scale) * np.sqrt(sum((a.astype(np.float64) ** 2).sum() for a in arrays))
        f = scale * limit / norm if norm > limit else (scale if norm == norm else np.nan)
        return norm, f, [a.astype(np.float64) * f for a in arrays]


def clip_check(api, got_norm, got, arrays, scale, limit, out_dtypes):
    """squares of floats are summed in double; those of halfs exactly squared in float, 8 at a
    time: 8 u relative, half of that in the norm. The factor is rounded to float, the product
    once, the result once."""
    norm, f, want = clip_formula(arrays, scale, limit)
    u = 2.0 ** -24
    rel = 4 * u + u + 1e-13
    close(got_norm, norm, 1.01 * rel * norm if np.isfinite(norm) else 0, "norm")
    for g, w, d in zip(got, want, out_dtypes):
        with np.errstate(all="ignore"):
            tol = 1.01 * np.abs(w) * (rel + 2 * u + U[np.dtype(d)]) + TINY[np.dtype(d)]
        close(g, w, np.where(np.isfinite(tol), tol, 0))


LISTS = [
    [(1,)], [(0,)], [], [(5,), (0, 3), ()], [(1000,), (3, 7), (1,)], [(8192,), (8193,), (16400,), (2,)], [(3,)] * 40, [(17,)] * 130,
]


@pytest.mark.parametrize("shapes", LISTS, ids=lambda s: "%d arrays" % len(s))
@pytest.mark.parametrize("dtype,out_dtype", [("f2", "f2"), ("f4", "f4"), ("f2", "f4"), ("f8", "f8")])
@pytest.mark.parametrize("limit", [0.5, INF, 0.0])
def test_clip(api, ctx, rng, shapes, dtype, out_dtype, limit):
    arrays = [rng.standard_normal(s).astype(dtype) for s in shapes]
    op = api.GpuClipNorm(ctx)
    src = [api.GpuArray.from_numpy(ctx, a) for a in arrays]
    dst = [api.GpuArray.from_numpy(ctx, np.full(s, 3, out_dtype)) for s in shapes]
    norm = api.GpuArray.empty(ctx, (), np.float32)
    op(norm, dst, src, limit, scale=0.5)
    first = [d.to_numpy() for d in dst]
    clip_check(api, norm.to_numpy(), first, arrays, 0.5, limit, [out_dtype] * len(arrays))
    op(norm, dst, src, limit, scale=0.5)               # the same bits again
    assert all((a == b.to_numpy()).all() for a, b in zip(first, dst))
    double = api.GpuArray.empty(ctx, (), np.float64)
    op(double, None, src, limit, scale=-0.5)           # the norm alone
    clip_check(api, double.to_numpy(), [], arrays, 0.5, limit, [])
    if dtype == out_dtype:
        op(norm, src, src, limit, scale=0.5)           # in place
        assert all((a == b.to_numpy()).all() for a, b in zip(first, src))
        assert all((a == b.to_numpy()).all() for a, b in zip(first, dst))


def test_clip_mixed_types_alignments_and_orders(api, ctx, rng):
    op = api.GpuClipNorm(ctx)
    arrays, src, dst, outs = [], [], [], []
    for i, (n, t, o) in enumerate([(300, "f2", "f4"), (301, "f4", "f4"), (77, "f8", "f8"), (2100, "f2", "f2"), (9, "f2", "f4")]):
        for k in (0, 1, 3, 5):
            a = rng.standard_normal(n).astype(t)
            arrays.append(a)
            src.append(at_offset(api, ctx, a, k))
            dst.append(at_offset(api, ctx, np.zeros(n, o), (k + i) % 4))
            outs.append(o)
    a = np.asfortranarray(rng.standard_normal((6, 11)).astype(np.float32))
    arrays.append(a)
    src.append(api.GpuArray.from_numpy(ctx, a, "F"))
    dst.append(api.GpuArray.empty(ctx, (6, 11), np.float32, "F"))
    outs.append("f4")
    norm = api.GpuArray.empty(ctx, (), np.float64)
    op(norm, dst, src, 1.0)
    clip_check(api, norm.to_numpy(), [d.to_numpy() for d in dst], arrays, 1.0, 1.0, outs)


def test_clip_infinities_nans_and_the_range_of_float(api, ctx, rng):
    op = api.GpuClipNorm(ctx)
    norm = api.GpuArray.empty(ctx, (), np.float64)
    for values, limit in (([3e38, 3e38, -1e38], 1.0), ([1e-30, 2e-30], 1e-30), ([1.0, np.nan], 1.0), ([1.0, INF], 1.0), ([1.0, INF], INF), ([0.0, 0.0], 0.0)):
        a = np.array(values, np.float32)
        dst = api.GpuArray.empty(ctx, a.shape, np.float32)
        op(norm, [dst], [put(api, ctx, a)], limit)
        clip_check(api, norm.to_numpy(), [dst.to_numpy()], [a], 1.0, limit, ["f4"])


@pytest.mark.parametrize("values,times,limit,scale", [
    ([1e38], 4, 1e-3, 1.0), ([1e38], 4, 1e-6, 1.0), ([1e38], 4, 1e-9, 1.0), ([3e38, -1e38, 2e30], 700, 1e-6, 1.0),
    ([3e38, 1.0], 1, INF, 1e-40), ([1e-38, -3e-39], 1, INF, 1e39), ([1e-44, 0.0], 1, 1e-3, 1e45)])
@pytest.mark.parametrize("in_place", [False, True])
def test_clip_factors_outside_the_range_of_float(api, ctx, values, times, limit, scale, in_place):
    """a factor that no normal float holds, between inputs and results that are floats. Its product
    is taken in double: the norm's error, one rounding to double and one to float are left"""
    a = np.array(values * times, np.float32)
    src, norm = put(api, ctx, a), api.GpuArray.empty(ctx, (), np.float64)
    dst = src if in_place else api.GpuArray.empty(ctx, a.shape, np.float32)
    api.GpuClipNorm(ctx)(norm, [dst], [src], limit, scale=scale)
    want_norm, f, want = clip_formula([a], scale, limit)
    assert np.isfinite(want[0]).all() and want[0].any() and not 2.0 ** -126 <= abs(f) < 2.0 ** 128
    close(norm.to_numpy(), want_norm, 1e-13 * want_norm, "norm")
    close(dst.to_numpy(), want[0], 1.01 * 2.0 ** -24 * np.abs(want[0]) + 2.0 ** -150)


def test_clip_of_halfs_by_a_factor_below_the_floats(api, ctx):
    """halfs into floats: results are floats although the factor is not a normal one"""
    a = np.array([60000.0, -0.25, 6e-8, 1000.0] * 3, np.float16)
    dst, norm = api.GpuArray.empty(ctx, a.shape, np.float32), api.GpuArray.empty(ctx, (), np.float64)
    api.GpuClipNorm(ctx)(norm, [dst], [put(api, ctx, a)], 1e-35)
    want_norm, f, want = clip_formula([a], 1.0, 1e-35)
    # squares of 8 halfs are summed in float: at most 8 half steps of the sum, half of that in the norm
    close(norm.to_numpy(), want_norm, 1.01 * 4 * 2.0 ** -24 * want_norm, "norm")
    close(dst.to_numpy(), want[0], 1.01 * 5 * 2.0 ** -24 * np.abs(want[0]) + 2.0 ** -150)


def test_clip_where_scale_and_norm_leave_the_doubles(api, ctx):
    """|scale| times the norm, or the limit over it, may be no double: dst is +-limit / |src| all the same"""
    op, norm = api.GpuClipNorm(ctx), api.GpuArray.empty(ctx, (), np.float64)
    for scale, limit in ((1e300, 1e-200), (-1e300, 2.0), (1e300, 1e300)):
        a = np.array([3.0, 4e20], np.float64)
        dst = api.GpuArray.empty(ctx, a.shape, np.float64)
        op(norm, [dst], [put(api, ctx, a)], limit, scale=scale)
        want = np.sign(scale) * a / np.sqrt((a * a).sum()) * limit
        close(dst.to_numpy(), want, 8 * 2.0 ** -53 * np.abs(want))


def test_clip_leaves_what_need_not_change(api, ctx, rng):
    """in place below the limit: the same bits; between arrays: untouched"""
    a = rng.standard_normal(1000).astype(np.float32)
    whole = put(api, ctx, a)
    parts = [whole[3:500], whole[600:999]]
    op = api.GpuClipNorm(ctx)
    norm = api.GpuArray.empty(ctx, (), np.float32)
    op(norm, parts, parts, 1e6)
    assert (whole.to_numpy() == a).all()
    op(norm, parts, parts, 1.0)
    got = whole.to_numpy()
    assert (got[:3] == a[:3]).all() and (got[500:600] == a[500:600]).all() and got[999] == a[999]
    assert abs(np.sqrt((got[3:500].astype(np.float64) ** 2).sum() + (got[600:999].astype(np.float64) ** 2).sum()) - 1) < 1e-6


# ------------------------------------------------------------------- all of them

def bigram_step(api, ctx, table, tokens, ops, buf, limit, entropy_weight):
    """one step of a bigram model: logits = rows of a V x V table, the loss and its gradient, the
    gradient of the table, clipped"""
    inputs, targets = tokens[:, :-1], tokens[:, 1:]
    api.embed(buf["logits"], table, inputs, scale=1.25, pad=0)
    ops["lp"](buf["logits"], targets, logp=buf["logp"], entropy=buf["ent"], stats=buf["stats"], ignore=0)
    ops["lp"].grad(buf["logits"], buf["logits"], targets, buf["stats"], buf["dlogp"], entropy=buf["ent"], dentropy=buf["dent"], ignore=0)
    ops["eg"](buf["dtable"], buf["logits"], inputs, scale=1.25, pad=0)
    ops["cn"](buf["norm"], [buf["dtable"]], [buf["dtable"]], limit)


def bigram_setup(api, ctx, rng, V, B, S, entropy_weight):
    table = (rng.standard_normal((V, V)) * 0.5).astype(np.float32)
    tokens = rng.integers(0, V, (B, S + 1)).astype(np.int32)
    ops = {"lp": api.GpuLogProbs(ctx, np.float32, np.int32), "eg": api.GpuEmbedGrad(ctx), "cn": api.GpuClipNorm(ctx)}
    f, e = np.float32, api.GpuArray.empty
    buf = {"logits": e(ctx, (B, S, V), f), "logp": e(ctx, (B, S), f), "ent": e(ctx, (B, S), f), "stats": e(ctx, (B, S, 2), f),
           "dlogp": put(api, ctx, np.full((B, S), -1.0, f)), "dent": put(api, ctx, np.full((B, S), -entropy_weight, f)),
           "dtable": e(ctx, (V, V), f), "norm": e(ctx, (), f)}
    return table, tokens, ops, buf


def bigram_formula(table, tokens, entropy_weight, limit):
    x, t = tokens[:, :-1], tokens[:, 1:]
    logits = embed_formula(table, x, 1.25, 0)
    logp, ent, _, _, _ = lp_formula(logits, t, 1.0, 0)
    g, _, _, _ = lp_grad_formula(logits, t, 1.0, -np.ones(t.shape), -entropy_weight * np.ones(t.shape), 0)
    dt, _, _ = grad_formula(table.shape[0], g, x, 1.25, 0)
    norm = np.sqrt((dt ** 2).sum())
    return logp, ent, dt * min(1, limit / norm), norm


def test_the_operators_together_make_a_training_step(api, ctx, rng):
    V, B, S = 37, 3, 9
    table, tokens, ops, buf = bigram_setup(api, ctx, rng, V, B, S, 0.1)
    gt = put(api, ctx, table)
    bigram_step(api, ctx, gt, put(api, ctx, tokens), ops, buf, 1.0, 0.1)
    logp, ent, dt, norm = bigram_formula(table, tokens, 0.1, 1.0)
    # the operators' own bounds, at these sizes all below 1e-5 of values of at most 10
    close(buf["logp"].to_numpy(), logp, 1e-4)
    close(buf["ent"].to_numpy(), ent, 1e-4)
    close(buf["norm"].to_numpy(), norm, 1e-4 * norm)
    close(buf["dtable"].to_numpy(), dt, 1e-4)


# ---------------------------------------------------------------------- refusals

def refused(api, code, call):
    with pytest.raises(api.GpuArrayException) as e:
        call()
    assert e.value.code == code, (e.value.code, str(e.value))


def test_embed_refusals(api, ctx):
    e = api.GpuArray.empty
    out, table, ids = e(ctx, (4, 8), np.float32), e(ctx, (5, 8), np.float32), put(api, ctx, np.zeros(4, np.int64))
    op = api.GpuEmbedGrad(ctx)
    for call in (lambda o, t, i: api.embed(o, t, i), lambda o, t, i: op(t, o, i)):
        call(out, table, ids)
        refused(api, api.GA_UNSUPPORTED_ERROR, lambda: call(out, table, put(api, ctx, np.zeros(4, np.int16))))
        refused(api, api.GA_UNSUPPORTED_ERROR, lambda: call(out, table, put(api, ctx, np.zeros(4, np.float32))))
        refused(api, api.GA_UNSUPPORTED_ERROR, lambda: call(e(ctx, (4, 8), np.int32), table, ids))
        refused(api, api.GA_UNSUPPORTED_ERROR, lambda: call(out, e(ctx, (5, 8), np.uint8), ids))
        refused(api, api.GA_VALUE_ERROR, lambda: call(e(ctx, (4, 7), np.float32), table, ids))
        refused(api, api.GA_VALUE_ERROR, lambda: call(e(ctx, (3, 8), np.float32), table, ids))
        refused(api, api.GA_VALUE_ERROR, lambda: call(e(ctx, (8,), np.float32), table, ids))
        refused(api, api.GA_VALUE_ERROR, lambda: call(out, e(ctx, (5, 8, 1), np.float32), ids))
    for bad in (INF, float("nan"), 1e300):
        refused(api, api.GA_VALUE_ERROR, lambda: api.embed(out, table, ids, scale=bad))
        refused(api, api.GA_VALUE_ERROR, lambda: op(table, out, ids, scale=bad))
    # a destination whose elements share places, one that may not be written, one beyond its buffer
    shared = api.GpuArray.from_pointer(ctx, out.devptr, (4, 8), np.float32, strides=(0, 4))
    refused(api, api.GA_VALUE_ERROR, lambda: api.embed(shared, table, ids))
    fixed = api.GpuArray.from_pointer(ctx, out.devptr, (4, 8), np.float32, writeable=False)
    refused(api, api.GA_VALUE_ERROR, lambda: api.embed(fixed, table, ids))
    refused(api, api.GA_VALUE_ERROR, lambda: op(fixed, table[:4], ids))
    beyond = api.GpuArray.from_pointer(ctx, out.devptr, (4, 8), np.float32, strides=(64, 4), nbytes=128)
    refused(api, api.GA_VALUE_ERROR, lambda: api.embed(beyond, table, ids))
    # a wrapped pointer between two elements
    odd = api.GpuArray.from_pointer(ctx, out.devptr + 2, (3, 8), np.float32)
    refused(api, api.GA_UNALIGNED_ERROR, lambda: api.embed(odd, table, ids[:3]))
    refused(api, api.GA_UNALIGNED_ERROR, lambda: op(table, odd, ids[:3]))
    refused(api, api.GA_UNALIGNED_ERROR, lambda: api.GpuLogProbs(ctx, np.float32)(odd, stats=e(ctx, (3, 2), np.float32)))
    refused(api, api.GA_UNALIGNED_ERROR, lambda: api.GpuClipNorm(ctx)(e(ctx, (), np.float32), [odd], [odd], 1.0))
    refused(api, api.GA_INVALID_ERROR, lambda: api.embed(out, None, ids))
    L = api.lib()
    assert L.GpuArray_embed(out.at, table.at, ids.at, 1.0, 0, 64) == api.GA_INVALID_ERROR
    assert L.GpuArray_embed(None, table.at, ids.at, 1.0, 0, 0) == api.GA_INVALID_ERROR


def test_pad_and_ignore_of_unsigned_ids_are_compared_by_their_bits(api, ctx):
    """-1 names the id 2^64 - 1, and no id of 32 bits"""
    f, e = np.float32, api.GpuArray.empty
    table, z = put(api, ctx, np.ones((3, 4), f)), put(api, ctx, np.zeros((2, 4), f))
    for t, padded in ((np.uint64, True), (np.uint32, False)):
        ids = put(api, ctx, np.array([2, np.iinfo(t).max], t))
        out, lp = put(api, ctx, np.full((2, 4), 5, f)), e(ctx, (2,), f)
        api.embed(out, table, ids, pad=-1)
        assert (out.to_numpy() == [[1] * 4, [0 if padded else 5] * 4]).all()
        api.GpuLogProbs(ctx, f, t)(z, ids, logp=lp, ignore=-1)
        assert lp.to_numpy()[1] == 0 if padded else np.isnan(lp.to_numpy()[1])


def test_embed_and_logprobs_refuse_more_than_four_dimensions_apart(api, ctx):
    """dimensions that lie one behind the other in all arrays count as one: four may be left"""
    e, f = api.GpuArray.empty, np.float32
    U = api.GA_UNSUPPORTED_ERROR
    for nd in (4, 5):
        shape = (2,) * nd
        inner = tuple(slice(0, 2) for _ in shape)
        for gaps in (False, True):
            ids = put(api, ctx, np.ones((3,) * nd, np.int32))[inner] if gaps else put(api, ctx, np.ones(shape, np.int32))
            rows, table = e(ctx, shape + (4,), f), put(api, ctx, np.ones((3, 4), f))
            lp = e(ctx, shape, f)
            for call in (lambda: api.embed(rows, table, ids), lambda: api.GpuLogProbs(ctx, f, np.int32)(rows, ids, logp=lp),
                         lambda: api.GpuEmbedGrad(ctx)(table, rows, ids)):
                if nd == 5 and gaps:
                    refused(api, U, call)
                else:
                    call()
            if not (nd == 5 and gaps):
                assert (rows.to_numpy() == 1).all() and (np.abs(lp.to_numpy() + np.log(4)) < 1e-6).all()
                assert (table.to_numpy() == np.array([[0], [2 ** nd], [0]])).all()


def test_logprobs_refusals(api, ctx):
    e = api.GpuArray.empty
    f = np.float32
    refused(api, api.GA_UNSUPPORTED_ERROR, lambda: api.GpuLogProbs(ctx, np.float64))
    refused(api, api.GA_UNSUPPORTED_ERROR, lambda: api.GpuLogProbs(ctx, f, np.int16))
    refused(api, api.GA_VALUE_ERROR, lambda: api.GpuLogProbs(ctx, f, np.int64, top=33))
    op = api.GpuLogProbs(ctx, f, np.int64, top=4)
    z, t, lp = put(api, ctx, np.zeros((3, 9), f)), put(api, ctx, np.zeros(3, np.int64)), e(ctx, (3,), f)
    st, tv, ti = e(ctx, (3, 2), f), e(ctx, (3, 4), f), e(ctx, (3, 4), np.int64)
    op(z, t, logp=lp, stats=st, top_logp=tv, top_ids=ti)
    V = api.GA_VALUE_ERROR
    refused(api, V, lambda: op(z, t))
    refused(api, V, lambda: op(z, logp=lp))
    refused(api, V, lambda: op(z, t, stats=st))
    refused(api, V, lambda: op(put(api, ctx, np.zeros((3, 9), np.float16)), t, logp=lp))
    refused(api, V, lambda: op(z, put(api, ctx, np.zeros(3, np.int32)), logp=lp))
    refused(api, V, lambda: op(z, t[:2], logp=lp))
    refused(api, V, lambda: op(z, t, logp=e(ctx, (3,), np.float64)))
    refused(api, V, lambda: op(z, stats=e(ctx, (3, 3), f)))
    refused(api, V, lambda: op(z, top_logp=e(ctx, (3, 5), f)))
    refused(api, V, lambda: op(z, top_ids=e(ctx, (3, 4), np.int32)))
    refused(api, V, lambda: op(z[:, :3], top_logp=tv))                    # more than there are
    refused(api, V, lambda: op(put(api, ctx, np.zeros((3, 0), f)), stats=st))
    refused(api, V, lambda: op(e(ctx, (), f), stats=e(ctx, (2,), f)))
    refused(api, V, lambda: api.GpuLogProbs(ctx, f)(z, top_logp=tv))
    for bad in (0.0, -1.0, INF, float("nan"), 1e300):
        refused(api, V, lambda: op(z, t, logp=lp, scale=bad))
        refused(api, V, lambda: op.grad(z, z, t, st, lp, scale=bad))
    refused(api, V, lambda: op.grad(e(ctx, (3, 9), np.float16), z, t, st, lp))
    refused(api, V, lambda: op.grad(e(ctx, (3, 8), f), z, t, st, lp))
    refused(api, V, lambda: op.grad(z, z, t, st, lp, dentropy=lp))
    refused(api, V, lambda: op.grad(z, z, t, lp, lp))
    refused(api, api.GA_INVALID_ERROR, lambda: op.grad(z, z, None, st, lp))
    refused(api, api.GA_INVALID_ERROR, lambda: op.grad(z, z, t, st, None))
    huge = api.GpuArray.from_pointer(ctx, z.devptr, (1, 1 << 28), f, strides=(4, 0), nbytes=4)
    refused(api, api.GA_XLARGE_ERROR, lambda: op(huge, stats=e(ctx, (1, 2), f)))


def test_clip_refusals(api, ctx):
    e = api.GpuArray.empty
    f = np.float32
    op = api.GpuClipNorm(ctx)
    norm, a, b = e(ctx, (), f), put(api, ctx, np.ones(10, f)), e(ctx, (10,), f)
    op(norm, [b], [a], 1.0)
    V, I = api.GA_VALUE_ERROR, api.GA_INVALID_ERROR
    refused(api, V, lambda: op(e(ctx, (1,), f), [b], [a], 1.0))
    refused(api, V, lambda: op(e(ctx, (), np.float16), [b], [a], 1.0))
    for limit, scale in ((-1.0, 1.0), (float("nan"), 1.0), (1.0, INF), (1.0, float("nan"))):
        refused(api, V, lambda: op(norm, [b], [a], limit, scale=scale))
    refused(api, api.GA_UNSUPPORTED_ERROR, lambda: op(norm, None, [put(api, ctx, np.ones(3, np.int32))], 1.0))
    refused(api, V, lambda: op(norm, [e(ctx, (10,), np.float16)], [a], 1.0))
    refused(api, V, lambda: op(norm, [e(ctx, (2, 5), f)], [a], 1.0))
    refused(api, I, lambda: op(norm, None, [a[::2]], 1.0))
    refused(api, I, lambda: op(norm, [e(ctx, (3, 4), f, "F")], [e(ctx, (3, 4), f)], 1.0))
    # the same array twice, overlapping ones, a destination that is another's source
    op(norm, None, [a, a], 1.0)
    assert abs(float(norm.to_numpy()) - 20 ** 0.5) < 1e-6
    refused(api, V, lambda: op(norm, [a, a], [a, a], 1.0))
    refused(api, V, lambda: op(norm, [a[:6], a[5:]], [a[:6], a[5:]], 1.0))
    refused(api, V, lambda: op(norm, [b, a], [a, b], 1.0))
    refused(api, V, lambda: op(norm, [a[:8]], [a[2:]], 1.0))
    inside = api.GpuArray.from_pointer(ctx, a.devptr + 8, (), f, nbytes=4)
    refused(api, V, lambda: op(inside, [a], [a], 1.0))
    refused(api, V, lambda: op(inside, [b], [a], 1.0))
    op(norm, [a[:5], a[5:]], [a[:5], a[5:]], 1.0)
    with pytest.raises(ValueError):
        op(norm, [b], [a, b], 1.0)


def test_clip_refuses_a_norm_inside_a_source_without_destinations(api, ctx):
    e = api.GpuArray.empty
    f = np.float32
    op, a, b = api.GpuClipNorm(ctx), put(api, ctx, np.ones(10, f)), put(api, ctx, np.ones(3, f))
    for k in (0, 2, 9):
        inside = api.GpuArray.from_pointer(ctx, a.devptr + 4 * k, (), f, nbytes=4)
        for src in ([a], [b, a], [a, b, a], [a[k:], b]):
            refused(api, api.GA_VALUE_ERROR, lambda: op(inside, None, src, 1.0))
        op(inside, None, [b, a[:k], a[k + 1:]], 1.0)       # beside the sources, and one of no elements
        assert float(inside.to_numpy()) == np.sqrt(f(12))
        a.write(np.ones(10, f))
    wide = api.GpuArray.from_pointer(ctx, a.devptr + 24, (), np.float64, nbytes=8)
    refused(api, api.GA_VALUE_ERROR, lambda: op(wide, None, [a[7:]], 1.0))
    op(wide, None, [a[7:7], b[:0]], 1.0)                   # arrays without elements overlap nothing
    assert float(wide.to_numpy()) == 0
    a.write(np.ones(10, f))
    assert (a.to_numpy() == 1).all()


def test_arrays_of_another_context_are_refused(api, ctx):
    other = api.Context(0)
    f = np.float32
    out, table, ids = api.GpuArray.empty(ctx, (2, 4), f), put(api, other, np.zeros((3, 4), f)), put(api, ctx, np.zeros(2, np.int32))
    V = api.GA_VALUE_ERROR
    refused(api, V, lambda: api.embed(out, table, ids))
    refused(api, V, lambda: api.GpuEmbedGrad(ctx)(table, out, ids))
    refused(api, V, lambda: api.GpuLogProbs(ctx, f)(table, stats=api.GpuArray.empty(ctx, (3, 2), f)))
    refused(api, V, lambda: api.GpuClipNorm(ctx)(api.GpuArray.empty(ctx, (), f), None, [table], 1.0))
    del table
    other.close()
