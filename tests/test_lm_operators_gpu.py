"""The language-model operators on a B200: the cases of lm_operators_cases.py,
and what needs a device: large sizes, offsets beyond 32 bits, graphs, rows in
the last wave."""
import numpy as np
import pytest

from lm_operators_cases import *  # noqa: F401,F403
from lm_operators_cases import (bigram_formula, bigram_setup, bigram_step, close, embed_formula, grad_formula, grad_tol,
                                lp_formula, lp_grad_formula, lp_grad_tol, lp_tols, put, rows_of_logits, check_top)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f2", "f4"])
@pytest.mark.parametrize("rows,V,top", [(1, 131072, 32), (3, 131071, 20), (40, 50021, 5), (200, 32000, 1), (700, 9000, 0),
                                        (5, 200003, 0), (150, 65536, 20), (3000, 1000, 3)])
@pytest.mark.parametrize("kind", ["plain", "masked", "ties"])
def test_logprobs_large(api, ctx, rng, dtype, rows, V, top, kind):
    z = rows_of_logits(rng, rows, V, dtype, kind)
    targets = rng.integers(0, V, rows).astype(np.int32)
    op = api.GpuLogProbs(ctx, dtype, np.int32, top=top)
    e = api.GpuArray.empty
    d = {"logp": e(ctx, (rows,), "f4"), "entropy": e(ctx, (rows,), "f4"), "stats": e(ctx, (rows, 2), "f4")}
    if top:
        d["top_logp"], d["top_ids"] = e(ctx, (rows, top), "f4"), e(ctx, (rows, top), "i4")
    gz, gt = put(api, ctx, z), put(api, ctx, targets)
    op(gz, gt, check=True, **d)
    first = {n: x.to_numpy() for n, x in d.items()}
    op(gz, gt, **d)
    assert all((first[n].view(np.int32) == x.to_numpy().view(np.int32)).all() for n, x in d.items())
    logp, ent, logs, p, empty = lp_formula(z, targets, 1.0)
    tol, tol_ent, gap = lp_tols(z, 1.0, p)
    with np.errstate(invalid="ignore"):
        tg = np.take_along_axis(gap, targets[:, None].astype(np.int64), -1)[:, 0]
        close(first["logp"], logp, tol + 4 * 2.0 ** -24 * (tg + np.log(V)), "logp")
        close(first["entropy"], ent, tol_ent, "entropy")
    if top:
        ids = first["top_ids"].astype(np.int64)
        with np.errstate(invalid="ignore"):
            g = np.take_along_axis(gap, ids, -1)
        some = slice(0, None, max(1, rows // 50))
        check_top(api, z[some], top, first["top_logp"][some], ids[some], logs[some], (tol[:, None] + 4 * 2.0 ** -24 * (g + np.log(V)))[some], empty)
    a = rng.standard_normal(rows).astype("f4")
    dz = e(ctx, (rows, V), dtype)
    op.grad(dz, gz, gt, d["stats"], put(api, ctx, a), entropy=d["entropy"], dentropy=put(api, ctx, a))
    want, p, logs, h = lp_grad_formula(z, targets, 1.0, a.astype(np.float64), a.astype(np.float64))
    tol = lp_grad_tol(z, 1.0, p, logs, h, a, a, dtype)
    close(dz.to_numpy(), want, tol + U[np.dtype(dtype)] * (np.abs(want) + tol) + TINY[np.dtype(dtype)])


@pytest.mark.parametrize("tokens,rows,width,dtype", [(20000, 5000, 256, "f2"), (4097, 1, 40, "f4"), (70001, 17, 64, "f2"), (9000, 100000, 33, "f4")])
@pytest.mark.parametrize("accumulate", [False, True])
def test_embed_gradient_large(api, ctx, rng, tokens, rows, width, dtype, accumulate):
    dout = rng.standard_normal((tokens, width)).astype(dtype)
    ids = (rows * rng.random(tokens) ** 4).astype(np.int64)
    base = rng.standard_normal((rows, width)).astype(dtype)
    op = api.GpuEmbedGrad(ctx)
    gd, gi, got = put(api, ctx, dout), put(api, ctx, ids), []
    for _ in range(2):
        dt = put(api, ctx, base)
        op(dt, gd, gi, scale=0.25, accumulate=accumulate, check=True)
        got.append(dt.to_numpy())
    assert (got[0] == got[1]).all()
    want, size, counts = grad_formula(rows, dout, ids, 0.25, None, base if accumulate else None)
    close(got[0], want, grad_tol(want, size, counts, dtype, False))
    out = api.GpuArray.empty(ctx, (tokens, width), dtype)
    api.embed(out, put(api, ctx, base), gi, check=True)
    assert (out.to_numpy() == base[ids]).all()


def test_offsets_beyond_32_bits(api, ctx):
    """a table, logits and gradients of more than 4 GiB (one byte offset in them passes 2^32), the
    last rows of each"""
    rows, width = 1 << 20, 2304                        # halfs: 4.5 GiB
    table = api.GpuArray.empty(ctx, (rows, width), "f2")
    table.memset(0)
    mark = np.arange(width).astype("f2") / 8
    table[rows - 1:].write(mark[None])
    ids = put(api, ctx, np.array([rows - 1, 0, -1], np.int64))
    out = api.GpuArray.empty(ctx, (3, width), "f2")
    api.embed(out, table, ids, check=True)
    got = out.to_numpy()
    assert (got[0] == mark).all() and (got[1] == 0).all() and (got[2] == mark).all()
    op = api.GpuEmbedGrad(ctx)
    op(table, out, ids, check=True)
    assert (table[rows - 2:].to_numpy() == np.stack([0 * mark, 2 * mark])).all()
    # the same memory as logits: (rows, width), only the last rows looked at
    t = api.GpuArray.empty(ctx, (rows,), np.int32)
    t.memset(0)
    lp = api.GpuLogProbs(ctx, "f2", np.int32)
    logp, stats = api.GpuArray.empty(ctx, (rows,), "f4"), api.GpuArray.empty(ctx, (rows, 2), "f4")
    lp(table, t, logp=logp, stats=stats, scale=0.01)
    z = np.stack([0 * mark, 2 * mark])
    want, _, _, p, _ = lp_formula(z, np.zeros(2, np.int64), 0.01)
    close(logp[rows - 2:].to_numpy(), want, 1e-4)
    lp.grad(table, table, t, stats, logp, scale=0.01)
    a = logp[rows - 2:].to_numpy().astype(np.float64)
    hot = np.zeros((2, width))
    hot[:, 0] = 1
    g = 0.01 * a[:, None] * (hot - p)
    close(table[rows - 2:].to_numpy(), g, np.abs(g) * (2.0 ** -11 + 1e-4) + 2.0 ** -24)


def test_training_steps_replay_from_a_graph(api, ctx, rng):
    """the operators captured together, replayed on new contents; a second graph with operators of
    its own over other sizes between the replays, and eager calls that make a workspace grow"""
    torch = pytest.importorskip("torch")
    stream = torch.cuda.ExternalStream(ctx.stream, device=0)
    steps = []
    for V, B, S in ((200, 4, 300), (90, 2, 70)):   # sorted tokens, and few
        table, tokens, ops, buf = bigram_setup(api, ctx, rng, V, B, S, 0.05)
        gt, gk = put(api, ctx, table), put(api, ctx, tokens)
        bigram_step(api, ctx, gt, gk, ops, buf, 0.5, 0.05)
        ctx.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            bigram_step(api, ctx, gt, gk, ops, buf, 0.5, 0.05)
        steps.append((V, B, S, ops, buf, gt, gk, graph))
    for trial in range(3):
        news = []
        for V, B, S, ops, buf, gt, gk, graph in steps:
            table = (rng.standard_normal((V, V)) * 0.5).astype("f4")
            tokens = rng.integers(0, V, (B, S + 1)).astype("i4")
            gt.write(table)
            gk.write(tokens)
            news.append((table, tokens))
        ctx.sync()
        for s in steps:
            s[7].replay()
        torch.cuda.synchronize()
        for (V, B, S, ops, buf, gt, gk, graph), (table, tokens) in zip(steps, news):
            logp, ent, dt, norm = bigram_formula(table, tokens, 0.05, 0.5)
            close(buf["logp"].to_numpy(), logp, 1e-4)
            close(buf["norm"].to_numpy(), norm, 1e-4 * norm)
            close(buf["dtable"].to_numpy(), dt, 1e-4)
        # the operator of a captured graph used eagerly on more: what the graph refers to is kept
        big = rng.integers(0, 50, 3000 * (trial + 1)).astype("i4")
        up = rng.standard_normal((big.size, 16)).astype("f4")
        dt = api.GpuArray.empty(ctx, (50, 16), "f4")
        steps[0][3]["eg"](dt, put(api, ctx, up), put(api, ctx, big))
        want, size, counts = grad_formula(50, up, big, 1.0, None)
        close(dt.to_numpy(), want, grad_tol(want, size, counts, "f4", False))


def test_clip_many_and_large(api, ctx, rng):
    """more arrays than one table holds, and arrays of many blocks"""
    op = api.GpuClipNorm(ctx)
    for n, size in ((2500, 37), (3, 3000017), (129, 5000)):
        flat = rng.standard_normal(n * size).astype("f4")
        whole, to = put(api, ctx, flat), api.GpuArray.empty(ctx, (n * size,), "f4")
        norm = api.GpuArray.empty(ctx, (), np.float64)
        op(norm, [to[i * size:(i + 1) * size] for i in range(n)], [whole[i * size:(i + 1) * size] for i in range(n)], 2.0)
        want = np.sqrt((flat.astype(np.float64) ** 2).sum())
        assert abs(float(norm.to_numpy()) - want) <= 1e-12 * want
        close(to.to_numpy(), flat * (2.0 / want), np.abs(flat) * (2.0 / want) * 4 * 2.0 ** -24)


def test_two_contexts_side_by_side(api, ctx, rng):
    """the operators on two contexts (two streams) of one device, their calls interleaved and
    nothing waited for in between"""
    other = api.Context(0, kernel_cache=None)
    work = []
    for c, V, B, S in ((ctx, 150, 3, 500), (other, 60, 5, 700)):
        table, tokens, ops, buf = bigram_setup(api, c, rng, V, B, S, 0.05)
        work.append((c, table, tokens, ops, buf, put(api, c, table), put(api, c, tokens)))
    for _ in range(5):
        for c, table, tokens, ops, buf, gt, gk in work:
            bigram_step(api, c, gt, gk, ops, buf, 0.5, 0.05)
    for c, table, tokens, ops, buf, gt, gk in work:
        logp, ent, dt, norm = bigram_formula(table, tokens, 0.05, 0.5)
        close(buf["logp"].to_numpy(), logp, 1e-4)
        close(buf["norm"].to_numpy(), norm, 1e-4 * norm)
        close(buf["dtable"].to_numpy(), dt, 1e-4)
    del work, c, ops, buf, gt, gk
    other.close()
