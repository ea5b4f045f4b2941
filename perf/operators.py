"""What the operators for language models are measured on.

Five kinds of calls, the memory-bound ends of a language model's step, as a user
of this library makes them on arrays that live on the GPU:

  lookup  token embedding: rows of a table by token id, times a scale
  scatter the table's gradient: the rows of an upstream gradient summed by id
  score   log probabilities of given tokens, entropy, the most likely alternatives
  train   log probabilities and entropy, and the gradient of both for the logits
  clip    the norm over all gradients of a step, and the gradients scaled by it

`run` computes them either in plain torch operations in 32 bits (`own` false)
or through libgpuarray_b200 (`own` true). Token ids follow a 1/rank law, as
words do; logits are normal with a few columns raised, as a trained model's are.
"""
import math
import os

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"half": torch.float16, "float": torch.float32}
IDS = {"int": torch.int32, "long": torch.int64}
_context = []


def listed():
    return [
        # a decode step of five sequences: latency
        dict(name="lookup 5 tokens", kind="lookup", batch=5, length=1, width=2048, rows=32000, type="half", ids="long", scale=1.0, pad=False),
        # the inputs of a training batch, tokens[:, :-1] of a longer array, scaled by sqrt(width)
        dict(name="lookup 4x4095", kind="lookup", batch=4, length=4095, width=4096, rows=65536, type="half", ids="int", scale=64.0, pad=False),
        # a fine-tuning batch with a small vocabulary
        dict(name="scatter 300 float", kind="scatter", batch=3, length=100, width=768, rows=1000, type="float", ids="long", scale=1.0, pad=True, steps=1),
        # two micro-batches accumulated into one gradient, an odd width
        dict(name="scatter 2x8190 float", kind="scatter", batch=2, length=4095, width=1021, rows=50021, type="float", ids="int", scale=1.0, pad=False, steps=2),
        # a whole training batch on a large table
        dict(name="scatter 32760 half", kind="scatter", batch=8, length=4095, width=2048, rows=128000, type="half", ids="long", scale=45.25, pad=True, steps=1),
        # a decode step of three sequences that reports 20 alternatives
        dict(name="score 3x131072 top 20", kind="score", rows=3, vocab=131072, type="half", ids="long", top=20, entropy=True, scale=1.25, mask=False),
        # scoring a prompt: odd rows start off the alignment of a vector
        dict(name="score 2047x50021 top 5", kind="score", rows=2047, vocab=50021, type="half", ids="int", top=5, entropy=False, scale=1.0, mask=True),
        # this library's benchmark shape, with entropy
        dict(name="score 16384x32000 float", kind="score", rows=16384, vocab=32000, type="float", ids="int", top=0, entropy=True, scale=1.0, mask=False),
        # a small model's training step
        dict(name="train 129x1000 float", kind="train", batch=3, length=43, vocab=1000, type="float", ids="int", entropy=False, scale=1.0, mask=False),
        # policy-gradient training with an entropy term, masked columns, ignored rows
        dict(name="train 4092x65536 half", kind="train", batch=4, length=1023, vocab=65536, type="half", ids="long", entropy=True, scale=0.8, mask=True),
        # a small model's gradients
        dict(name="clip 24 small", kind="clip", layers=3, width=100, vocab=1000, type="float", out="float", scale=1.0),
        # a larger one's: half gradients under a loss scale, clipped into float for the optimiser
        dict(name="clip 52 half", kind="clip", layers=7, width=1600, vocab=50021, type="half", out="float", scale=1.0 / 1024),
    ]


def _spread(rng, lo, hi):
    """a whole number between lo and hi, spread over its logarithm"""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["lookup", "scatter", "score", "train", "clip"])
    kind_of = dict(type=rng.choice(["half", "float"]), ids=rng.choice(["int", "long"]))
    scale = rng.choice([1.0, round(rng.uniform(0.5, 2.0), 3)])
    if kind in ("lookup", "scatter"):
        width, rows = _spread(rng, 32, 4096), _spread(rng, 50, 131072)
        width = min(width, max(32, 200_000_000 // rows))
        batch, length = rng.randint(1, 8), _spread(rng, 1, 4096)
        length = min(length, max(1, 70_000_000 // (batch * width)))
        c = dict(kind=kind, batch=batch, length=length, width=width, rows=rows, scale=scale, pad=rng.random() < 0.5, **kind_of)
        return dict(c, steps=rng.choice([1, 1, 2])) if kind == "scatter" else c
    if kind == "score":
        vocab = _spread(rng, 40, 131072)
        rows = _spread(rng, 1, max(1, min(16384, 250_000_000 // vocab)))
        return dict(kind=kind, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 20]), entropy=rng.random() < 0.5, scale=scale, mask=rng.random() < 0.5, **kind_of)
    if kind == "train":
        vocab = _spread(rng, 40, 131072)
        batch = rng.randint(1, 4)
        length = _spread(rng, 1, max(1, min(4096, 200_000_000 // (vocab * batch))))
        return dict(kind=kind, batch=batch, length=length, vocab=vocab, entropy=rng.random() < 0.5, scale=scale, mask=rng.random() < 0.5, **kind_of)
    out = "float" if kind_of["type"] == "float" else rng.choice(["half", "float"])
    return dict(kind=kind, layers=rng.randint(1, 7), width=_spread(rng, 16, 1600), vocab=_spread(rng, 100, 50021), type=kind_of["type"], out=out, scale=rng.choice([1.0, 1.0 / 1024]))


def _sizes(c):
    """a model's parameters: per layer four products, two biases and a norm; an embedding and two norms"""
    w = c["width"]
    layer = [(w, 3 * w), (3 * w,), (w, w), (w, 4 * w), (4 * w,), (4 * w, w), (w,)]
    return [shape for _ in range(c["layers"]) for shape in layer] + [(c["vocab"], w), (w,), (w,)]


def _distinct(rows, tokens):
    """how many rows of a table `tokens` draws by the 1/rank law are expected to name"""
    r = np.arange(1, rows + 1, dtype=np.float64)
    p = np.log((r + 1) / r) / math.log(rows + 1)
    return float(np.sum(-np.expm1(tokens * np.log1p(-np.minimum(p, 1 - 1e-12)))))


def work(case):
    c = case
    size = 2 if c.get("type") == "half" else 4
    id_size = 4 if c.get("ids") == "int" else 8
    if c["kind"] in ("lookup", "scatter"):
        tokens, row = c["batch"] * c["length"], c["width"] * size
        if c["kind"] == "lookup":
            return {"bytes": tokens * (row + id_size) + _distinct(c["rows"], tokens) * row, "flops": tokens * c["width"]}
        again = (c["steps"] - 1) * 2 * _distinct(c["rows"], tokens) * row
        return {"bytes": c["steps"] * tokens * (row + id_size) + c["rows"] * row + again, "flops": c["steps"] * 2 * tokens * c["width"]}
    if c["kind"] == "clip":
        n = sum(math.prod(s) for s in _sizes(c))
        return {"bytes": n * (size + (2 if c["out"] == "half" else 4)), "flops": 3 * n}
    rows = c["rows"] if c["kind"] == "score" else c["batch"] * c["length"]
    n = rows * c["vocab"]
    if c["kind"] == "score":
        return {"bytes": n * size + rows * (id_size + 4 + 4 * c["entropy"] + c["top"] * (4 + id_size)), "flops": (6 if c["entropy"] else 4) * n}
    return {"bytes": 2 * n * size + rows * (id_size + 16), "flops": (12 if c["entropy"] else 8) * n}


def _ids(g, shape, rows, dtype):
    """token ids by the 1/rank law, the ranks spread over the table"""
    u = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)
    rank = torch.clamp(torch.exp(u * math.log(rows + 1)).long() - 1, 0, rows - 1)
    return ((rank * 40503 + 17) % rows if math.gcd(rows, 40503) == 1 else rank).to(dtype)


def _logits(g, shape, c):
    """normal logits, one in 300 raised; with a mask a tenth of the columns of a row is -inf, and one row in 500 wholly"""
    z = torch.randn(shape, generator=g, device="cuda").mul_(2)
    z.add_(torch.rand(shape, generator=g, device="cuda").lt_(1 / 300), alpha=6)
    if c["mask"]:
        z.masked_fill_(torch.rand(shape, generator=g, device="cuda", dtype=torch.float16) < 0.1, -math.inf)
        z.masked_fill_((torch.rand(shape[:-1], generator=g, device="cuda") < 0.002).unsqueeze(-1), -math.inf)
    return z.to(TYPES[c["type"]])


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "clip":
        # the scale of a gradient differs from tensor to tensor; the norm is a few times the limit
        s["grads"] = [(torch.randn(shape, generator=g, device="cuda") * (0.2 + i % 5) / c["scale"] / 100).to(TYPES[c["type"]]) for i, shape in enumerate(_sizes(c))]
        s["limit"] = 1.0
    elif c["kind"] in ("lookup", "scatter"):
        dtype = TYPES[c["type"]]
        s["pad"] = 3 if c["pad"] else None
        s["tokens"] = [_ids(g, (c["batch"], c["length"] + 1), c["rows"], IDS[c["ids"]])[:, :-1] for _ in range(c.get("steps", 1))]
        if c["kind"] == "lookup":
            s["table"] = torch.randn((c["rows"], c["width"]), generator=g, device="cuda").mul_(0.05).to(dtype)
        else:
            s["upstream"] = [torch.randn((c["batch"], c["length"], c["width"]), generator=g, device="cuda").mul_(0.01).to(dtype) for _ in range(c["steps"])]
    else:
        lead = (c["rows"],) if c["kind"] == "score" else (c["batch"], c["length"])
        s["logits"] = _logits(g, lead + (c["vocab"],), c)
        s["targets"] = torch.randint(0, c["vocab"], lead[:-1] + (lead[-1] + 1,), generator=g, device="cuda")[..., 1:].to(IDS[c["ids"]])
        if c["kind"] == "train":
            s["targets"] = torch.where(torch.rand(lead, generator=g, device="cuda") < 0.05, -1, s["targets"])
            s["dlogp"] = torch.randn(lead, generator=g, device="cuda")
            s["dentropy"] = 0.05 * torch.rand(lead, generator=g, device="cuda") if c["entropy"] else None
    if own:
        _handles(s)
    torch.cuda.synchronize()
    return s


def _handles(s):
    """the library's arrays over the same memory, the outputs and the operators, as a user's program holds them"""
    from libgpuarray_b200 import api

    if not _context:
        _context.append(api.Context(0, kernel_cache=os.path.join(ROOT, ".kernel_cache")))
    ctx, c = _context[0], s["case"]
    numpy_of = {torch.float16: np.float16, torch.float32: np.float32, torch.int32: np.int32, torch.int64: np.int64}

    def array(t):
        return None if t is None else api.GpuArray.from_pointer(ctx, t.data_ptr(), t.shape, numpy_of[t.dtype], [k * t.element_size() for k in t.stride()])

    def new(shape, dtype):
        t = torch.zeros(shape, dtype=dtype, device="cuda")
        return t, array(t)

    out, h = {}, {"api": api}
    if c["kind"] == "clip":
        made = [new(x.shape, TYPES[c["out"]]) for x in s["grads"]]
        out["grads"], h["to"] = [t for t, _ in made], api.GpuArrayList([a for _, a in made])
        h["from"] = api.GpuArrayList([array(x) for x in s["grads"]])
        out["norm"], h["norm"] = new((), torch.float32)
        h["op"] = api.GpuClipNorm(ctx)
    elif c["kind"] in ("lookup", "scatter"):
        h["tokens"] = [array(t) for t in s["tokens"]]
        shape = (c["rows"], c["width"]) if c["kind"] == "scatter" else (c["batch"], c["length"], c["width"])
        out["out"], h["out"] = new(shape, TYPES[c["type"]])
        if c["kind"] == "scatter":
            h["upstream"], h["op"] = [array(t) for t in s["upstream"]], api.GpuEmbedGrad(ctx)
        else:
            h["table"] = array(s["table"])
    else:
        lead = s["targets"].shape
        h["logits"], h["targets"] = array(s["logits"]), array(s["targets"])
        out["logp"], h["logp"] = new(lead, torch.float32)
        h["entropy"] = None
        if c["entropy"]:
            out["entropy"], h["entropy"] = new(lead, torch.float32)
        h["top_logp"] = h["top_ids"] = None
        if c.get("top"):
            out["top_logp"], h["top_logp"] = new(lead + (c["top"],), torch.float32)
            out["top_ids"], h["top_ids"] = new(lead + (c["top"],), IDS[c["ids"]])
        if c["kind"] == "train":
            s["stats"], h["stats"] = new(lead + (2,), torch.float32)
            out["dlogits"], h["dlogits"] = new(s["logits"].shape, TYPES[c["type"]])
            h["dlogp"], h["dentropy"] = array(s["dlogp"]), array(s["dentropy"])
        h["op"] = api.GpuLogProbs(ctx, numpy_of[TYPES[c["type"]]], numpy_of[IDS[c["ids"]]], top=c.get("top", 0))
    s["out"], s["handles"] = out, h


def run(state):
    s = state
    if own:
        return _run_own(s)
    return {"lookup": _lookup, "scatter": _scatter, "score": _score, "train": _train, "clip": _clip}[s["case"]["kind"]](s)


def _run_own(s):
    c, h = s["case"], s["handles"]
    kind = c["kind"]
    if kind == "lookup":
        h["api"].embed(h["out"], h["table"], h["tokens"][0], scale=c["scale"], pad=s["pad"])
    elif kind == "scatter":
        h["op"](h["out"], h["upstream"][0], h["tokens"][0], scale=c["scale"], pad=s["pad"])
        if c["steps"] == 2:
            h["op"](h["out"], h["upstream"][1], h["tokens"][1], scale=c["scale"], pad=s["pad"], accumulate=True)
    elif kind == "score":
        h["op"](h["logits"], h["targets"], logp=h["logp"], entropy=h["entropy"], top_logp=h["top_logp"], top_ids=h["top_ids"], scale=c["scale"])
    elif kind == "train":
        h["op"](h["logits"], h["targets"], logp=h["logp"], entropy=h["entropy"], stats=h["stats"], scale=c["scale"], ignore=-1)
        h["op"].grad(h["dlogits"], h["logits"], h["targets"], h["stats"], h["dlogp"], entropy=h["entropy"], dentropy=h["dentropy"], scale=c["scale"], ignore=-1)
    else:
        h["op"](h["norm"], h["to"], h["from"], s["limit"], scale=c["scale"])
    return s["out"]


def _kept(ids, pad):
    return torch.ones_like(ids, dtype=torch.float32) if pad is None else (ids != pad).float()


def _lookup(s):
    """out[t] = scale * table[ids[t]], and zero where ids[t] is the padding id"""
    ids = s["tokens"][0]
    rows = s["table"][ids].float() * s["case"]["scale"]
    rows = rows * _kept(ids, s["pad"]).unsqueeze(-1) if s["pad"] is not None else rows
    return {"out": rows.to(s["table"].dtype)}


def _summed(s, k):
    ids, up = s["tokens"][k].reshape(-1), s["upstream"][k]
    rows = up.reshape(len(ids), -1).float() * s["case"]["scale"]
    rows = rows * _kept(ids, s["pad"]).unsqueeze(-1) if s["pad"] is not None else rows
    return torch.zeros((s["case"]["rows"], rows.shape[1]), device="cuda").index_add_(0, ids, rows)


def _scatter(s):
    """out[v] = scale * sum of upstream[t] over the tokens with ids[t] = v; a second micro-batch is added to the first"""
    dtype = s["upstream"][0].dtype
    out = _summed(s, 0).to(dtype)
    return {"out": out if s["case"]["steps"] == 1 else (out.float() + _summed(s, 1)).to(dtype)}


def _softmax(s):
    """x, exp(x - max), its sum, log-sum-exp and which rows have no finite logit (their log-sum-exp is -inf)"""
    x = s["logits"].float() * s["case"]["scale"]
    top = x.amax(-1)
    empty = top == -math.inf
    ref = torch.where(empty, 0.0, top)
    d = x - ref.unsqueeze(-1)
    e = torch.exp(d)
    total = e.sum(-1)
    return x, d, e, total, ref + torch.log(total), empty


def _logp(s, x, lse, empty):
    """the target's log probability: -inf in a row without a finite logit, 0 where the target is -1"""
    t = s["targets"].long()
    found = x.gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1) - lse
    return torch.where(t == -1, 0.0, torch.where(empty, -math.inf, found)) if s["case"]["mask"] or s["case"]["kind"] == "train" else found


def _entropy(d, e, total, empty):
    """log(sum e) - sum(e d) / sum(e), 0 in a row without a finite logit"""
    return torch.where(empty, 0.0, torch.log(total) - (e * torch.where(e > 0, d, 0.0)).sum(-1) / total)


def _score(s):
    c = s["case"]
    x, d, e, total, lse, empty = _softmax(s)
    out = {"logp": _logp(s, x, lse, empty)}
    if c["entropy"]:
        out["entropy"] = _entropy(d, e, total, empty)
    if c["top"]:
        # one whole number orders by value and, among equal values, by the lower index
        bits = (s["logits"].float() + 0.0).view(torch.int32)
        place = torch.arange(c["vocab"], device="cuda")
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) + ((1 << 32) - 1 - place)
        index = key.topk(c["top"], -1).indices
        top = x.gather(-1, index) - lse.unsqueeze(-1)
        out["top_logp"] = torch.where(empty.unsqueeze(-1), -math.inf, top)
        out["top_ids"] = index.to(s["targets"].dtype)
    return out


def _train(s):
    """dx_j = scale * (dlogp (1[j = target] - p_j) - dentropy p_j (log p_j + entropy)); 0 for a target of -1 and in a row without a finite logit"""
    c = s["case"]
    x, d, e, total, lse, empty = _softmax(s)
    out = {"logp": _logp(s, x, lse, empty)}
    kept = s["targets"] != -1
    w = torch.where(kept & ~empty, s["dlogp"], 0.0)
    p = e * (1 / torch.where(empty, 1.0, total)).unsqueeze(-1)
    grad = -w.unsqueeze(-1) * p
    if c["entropy"]:
        out["entropy"] = _entropy(d, e, total, empty)
        logp = d - torch.log(total).unsqueeze(-1)
        grad = grad - (s["dentropy"] * ~empty).unsqueeze(-1) * p * (torch.where(p > 0, logp, 0.0) + out["entropy"].unsqueeze(-1))
    grad.scatter_add_(-1, s["targets"].long().clamp(min=0).unsqueeze(-1), w.unsqueeze(-1))
    out["dlogits"] = (grad * c["scale"]).to(s["logits"].dtype)
    return out


def _clip(s):
    """norm = |scale * all gradients|, each gradient times scale * min(1, limit / norm)"""
    c = s["case"]
    squares = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]])
    norm = squares.sum().sqrt() * c["scale"]
    factor = (c["scale"] * torch.where(norm > s["limit"], s["limit"] / norm, 1.0)).float()
    return {"norm": norm.float(), "grads": [(g.float() * factor).to(TYPES[c["out"]]) for g in s["grads"]]}


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"] == "clip":
        grads = [g.double() * c["scale"] for g in s["grads"]]
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g) for g in grads]))
        return {"norm": norm, "grads": [g * min(1.0, s["limit"] / float(norm)) for g in grads]}
    if c["kind"] == "lookup":
        ids = s["tokens"][0].long()
        out = s["table"].double()[ids] * c["scale"]
        out[ids == (-1 if s["pad"] is None else s["pad"])] = 0
        return {"out": out}
    if c["kind"] == "scatter":
        out = torch.zeros(c["rows"], c["width"], dtype=torch.float64, device="cuda")
        for ids, up in zip(s["tokens"], s["upstream"]):
            keep = ids != (-1 if s["pad"] is None else s["pad"])
            out.index_put_((ids[keep].long(),), up[keep].double() * c["scale"], accumulate=True)
        return {"out": out}
    z = s["logits"].double() * c["scale"]
    t = s["targets"].long()
    logs = torch.log_softmax(z, -1)
    empty = torch.isneginf(z).all(-1)
    logs = torch.where(empty.unsqueeze(-1), -math.inf, logs)
    logp = torch.where(t < 0, 0.0, logs.gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1))
    p = logs.exp()
    entropy = torch.special.entr(p).sum(-1)
    out = {"logp": logp}
    if c["entropy"]:
        out["entropy"] = entropy
    if c.get("top"):
        out["top_logp"] = logs.sort(-1, descending=True).values[..., : c["top"]].clone()
        out["top_ids"] = None
    if c["kind"] == "train":
        hot = torch.zeros_like(p).scatter_(-1, t.clamp(min=0).unsqueeze(-1), 1.0)
        g = s["dlogp"].double().unsqueeze(-1) * (t >= 0).unsqueeze(-1) * (hot - p)
        if c["entropy"]:
            g = g - s["dentropy"].double().unsqueeze(-1) * (-torch.special.entr(p) + p * entropy.unsqueeze(-1))
        out["dlogits"] = torch.where(empty.unsqueeze(-1), 0.0, g) * c["scale"]
    return out
