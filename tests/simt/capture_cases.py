"""What the language-model operators refuse while the stream is captured: calls
that wait, and a workspace that would have to grow. The stand-in driver is told
that a capture is on."""
import ctypes

import numpy as np
import pytest


@pytest.fixture()
def capturing():
    f = ctypes.CDLL("libcuda.so.1").fake_cuda_set_capturing
    yield f
    f(0)


def put(api, ctx, a):
    return api.GpuArray.from_numpy(ctx, a)


def test_captured_calls(api, ctx, rng, capturing):
    table = put(api, ctx, rng.standard_normal((5, 8)).astype(np.float32))
    ids, more = put(api, ctx, np.array([1, 3], np.int32)), put(api, ctx, np.zeros(2500, np.int32))
    out, long = api.GpuArray.empty(ctx, (2, 8), np.float32), api.GpuArray.empty(ctx, (2500, 8), np.float32)
    t = put(api, ctx, np.array([1, 3], np.int64))
    logp, stats, dl = (api.GpuArray.empty(ctx, s, np.float32) for s in ((2,), (2, 2), (2,)))
    lp, eg = api.GpuLogProbs(ctx, np.float32), api.GpuEmbedGrad(ctx)

    def every(check):
        api.embed(out, table, ids, check=check)
        eg(table, out, ids, check=check)
        lp(out, t, logp=logp, stats=stats, check=check)
        lp.grad(out, out, t, stats, dl, check=check)
    every(False)
    eg(table, long[:1100], more[:1100])                  # sorted tokens: the workspace is made
    capturing(1)
    eg(table, long[:1100], more[:1100])
    every(False)                                       # a repeated call needs nothing new
    for call in (lambda: api.embed(out, table, ids, check=True), lambda: eg(table, out, ids, check=True),
                 lambda: lp(out, t, logp=logp, check=True), lambda: lp.grad(out, out, t, stats, dl, check=True),
                 lambda: eg(table, long, more)):       # a longer call: the workspace would grow
        with pytest.raises(api.GpuArrayException) as e:
            call()
        assert e.value.code == api.GA_UNSUPPORTED_ERROR
    capturing(0)
    eg(table, long, more)
    every(True)
