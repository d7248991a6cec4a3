"""Timed cases of the operators between a language model's matrix products: embedding lookup and its table's
gradient, layer norm and its gradients, log probabilities of given tokens and their gradient, and clipping by the
global norm. `run` computes them either from elementary torch operations or, with `own`, through the library."""
import math
import random

import torch

own = False

TYPES = {"float": torch.float32, "double": torch.float64, "half": torch.float16}
SIZES = {"float": 4, "double": 8, "half": 2}

_ops = None


def _wide(name):
    """The type that sums and statistics have."""
    return torch.float64 if name == "double" else torch.float32


def _listed_layer_norm():
    return [
        # one token of a decoding step
        {"name": "norm one token", "op": "layer_norm", "type": "half", "rows": 1, "cols": 4096},
        # the activations of a training batch, at the size of the elementwise chain's arrays
        {"name": "norm activations", "op": "layer_norm", "type": "float", "rows": 16384, "cols": 4096},
        # backward pass over many short rows
        {"name": "norm gradient", "op": "layer_norm_grad", "type": "float", "rows": 65536, "cols": 1024},
        # backward pass over rows of an odd width, none of them aligned to the next
        {"name": "norm gradient odd half", "op": "layer_norm_grad", "type": "half", "rows": 10007, "cols": 2047},
    ]


def _listed_log_probs():
    return [
        # the next token of eight sequences, with the twenty best alternatives
        {"name": "next token alternatives", "op": "log_probs", "type": "half", "rows": 8, "vocab": 131072, "k": 20},
        # scoring a batch of text
        {"name": "score a batch", "op": "log_probs", "type": "float", "rows": 4096, "vocab": 32768, "k": 0},
        # the loss' gradient over a vocabulary of odd size
        {"name": "loss gradient half", "op": "log_probs_grad", "type": "half", "rows": 8192, "vocab": 50001, "entropy": False},
        # a policy's gradient with an entropy bonus, in double precision
        {"name": "policy gradient double", "op": "log_probs_grad", "type": "double", "rows": 1021, "vocab": 20000, "entropy": True},
    ]


def _listed_embedding():
    return [
        # the tokens of a training batch
        {"name": "lookup", "op": "embedding", "type": "half", "tokens": 32768, "cols": 2048, "vocab": 100000},
        # their gradient, written over the whole table; a few tokens make up much of the text
        {"name": "table gradient", "op": "embedding_grad", "type": "float", "tokens": 16384, "cols": 1024, "vocab": 50000},
    ]


def _listed_clip():
    return [
        # the tensors of a small network
        {"name": "clip small", "op": "clip", "type": "float", "tensors": 40, "total": 200003, "clipped": True},
        # the gradients of a large one
        {"name": "clip large", "op": "clip", "type": "float", "tensors": 60, "total": 134217728, "clipped": True},
    ]


def listed():
    return _listed_layer_norm() + _listed_log_probs() + _listed_embedding() + _listed_clip()


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm_grad", "log_probs", "log_probs_grad", "embedding", "embedding_grad", "clip"])
    kind = rng.choice(["float", "float", "half", "half", "double"])
    size = SIZES[kind]
    if op in ("layer_norm", "layer_norm_grad"):
        cols = _spread(rng, 16, 16384)
        rows = _spread(rng, 1, min(65536, 700000000 // (3 * size * cols)))
        return {"op": op, "type": kind, "rows": rows, "cols": cols}
    if op == "log_probs":
        vocab = _spread(rng, 500, 150000)
        k = rng.choice([0, 0, 1, 5, 20, 32])
        rows = _spread(rng, 1, min(8192, (500000000 if k == 0 else 200000000) // (size * vocab)))
        return {"op": op, "type": kind, "rows": rows, "vocab": vocab, "k": k}
    if op == "log_probs_grad":
        vocab = _spread(rng, 500, 150000)
        rows = _spread(rng, 1, min(8192, 350000000 // (size * vocab)))
        return {"op": op, "type": kind, "rows": rows, "vocab": vocab, "entropy": rng.random() < 0.5}
    if op == "embedding":
        cols = _spread(rng, 64, 8192)
        return {"op": op, "type": kind, "tokens": _spread(rng, 1, min(65536, 300000000 // (size * cols))), "cols": cols,
                "vocab": _spread(rng, 500, min(150000, 400000000 // (size * cols)))}
    if op == "embedding_grad":
        cols = _spread(rng, 64, 8192)
        return {"op": op, "type": kind, "tokens": _spread(rng, 1, min(65536, 200000000 // (size * cols))), "cols": cols,
                "vocab": _spread(rng, 500, min(150000, 300000000 // (size * cols)))}
    total = _spread(rng, 1000, 400000000 // size)
    return {"op": "clip", "type": kind, "tensors": _spread(rng, 1, 60), "total": total, "clipped": rng.random() < 0.7}


def _lengths(case):
    """How the values are spread over the tensors: a few large matrices, many short vectors."""
    rng = random.Random(case["tensors"] * 1000003 + case["total"])
    weights = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(case["tensors"])]
    total = sum(weights)
    lengths = [int(case["total"] * w / total) for w in weights]
    lengths[0] += case["total"] - sum(lengths)
    return lengths


def _text(case, gen):
    """Tokens whose frequency falls with the inverse of their rank, the ranks scattered over the table."""
    n, vocab = case["tokens"], case["vocab"]
    rank = torch.pow(float(vocab), torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)).long() - 1
    tokens = torch.randperm(vocab, device="cuda", generator=gen)[rank.clamp_(0, vocab - 1)]
    tokens[torch.rand(n, device="cuda", generator=gen) < 0.02] = -1     # positions behind a sequence's end
    return tokens


def _prepare_layer_norm(case, gen):
    kind, rows, cols = TYPES[case["type"]], case["rows"], case["cols"]
    x = torch.randn(rows, cols, device="cuda", generator=gen) * 1.5
    x += 0.3 * torch.randn(rows, 1, device="cuda", generator=gen)      # the residual stream is not centred
    state = {"x": x.to(kind), "epsilon": 1e-5,
             "gain": (1 + 0.2 * torch.randn(cols, device="cuda", generator=gen)).to(kind),
             "bias": (0.1 * torch.randn(cols, device="cuda", generator=gen)).to(kind)}
    wide = state["x"].double()
    mean = wide.mean(1)
    state["mean"] = mean.to(_wide(case["type"]))
    state["invStd"] = (1 / torch.sqrt(((wide - mean[:, None]) ** 2).mean(1) + state["epsilon"])).to(_wide(case["type"]))
    if case["op"] == "layer_norm_grad":
        state["dz"] = torch.randn(rows, cols, device="cuda", generator=gen).to(kind)
    return state


def _prepare_log_probs(case, gen):
    kind, rows, vocab = TYPES[case["type"]], case["rows"], case["vocab"]
    logits = torch.randn(rows, vocab, device="cuda", generator=gen) * 2.5
    logits[:, vocab - vocab // 200:] = -math.inf                        # entries behind the vocabulary's end
    tokens = torch.randint(0, vocab - vocab // 200, (rows,), device="cuda", generator=gen)
    at = torch.arange(rows, device="cuda")
    logits[at, tokens] += 6.0 * torch.rand(rows, device="cuda", generator=gen)
    tokens[torch.rand(rows, device="cuda", generator=gen) < 0.04] = -1  # positions behind a sequence's end
    state = {"logits": logits.to(kind), "tokens": tokens, "scale": 0.8}
    if case["op"] == "log_probs_grad":
        wide = _wide(case["type"])
        x = state["logits"].double()
        top = x.amax(1)
        e = torch.exp((x - top[:, None]) * state["scale"])
        s = e.sum(1)
        x.sub_(top[:, None]).mul_(state["scale"]).nan_to_num_(neginf=0.0).mul_(e)
        state["rowMax"], state["logSum"] = top.to(wide), s.log().to(wide)
        state["entropy"] = (s.log() - x.sum(1) / s).to(wide)
        loss_scale = 65536.0 / rows
        state["dLogProbs"] = (-loss_scale * torch.rand(rows, device="cuda", generator=gen)).to(wide)
        state["dEntropy"] = (0.1 * loss_scale * torch.rand(rows, device="cuda", generator=gen)).to(wide) if case["entropy"] else None
    return state


def _prepare_embedding(case, gen):
    kind = TYPES[case["type"]]
    state = {"tokens": _text(case, gen), "scale": math.sqrt(case["cols"])}
    if case["op"] == "embedding":
        state["table"] = (0.02 * torch.randn(case["vocab"], case["cols"], device="cuda", generator=gen)).to(kind)
    else:
        state["scale"] = 0.25
        state["dz"] = torch.randn(case["tokens"], case["cols"], device="cuda", generator=gen).to(kind)
    return state


def _prepare_clip(case, gen):
    x = [(0.01 * torch.randn(n, device="cuda", generator=gen)).to(TYPES[case["type"]]) for n in _lengths(case)]
    expected = 0.01 * math.sqrt(case["total"])
    return {"x": x, "lengths": [t.numel() for t in x], "maxNorm": expected * (0.4 if case["clipped"] else 2.5)}


def _outputs(case, state):
    """The buffers that the library's calls write into."""
    kind, wide = TYPES[case["type"]], _wide(case["type"])
    rows = case.get("rows", 0)

    def new(shape, kind):
        return torch.empty(shape, device="cuda", dtype=kind)
    if case["op"] == "layer_norm":
        return [new((rows, case["cols"]), kind), new(rows, wide), new(rows, wide)]
    if case["op"] == "layer_norm_grad":
        return [new((rows, case["cols"]), kind), new(case["cols"], kind), new(case["cols"], kind)]
    if case["op"] == "log_probs":
        best = [new((rows, case["k"]), torch.int64), new((rows, case["k"]), wide)] if case["k"] else []
        return [new(rows, wide) for _ in range(4)] + best
    if case["op"] == "log_probs_grad":
        return [new((rows, case["vocab"]), kind)]
    if case["op"] == "embedding":
        return [new((case["tokens"], case["cols"]), kind)]
    if case["op"] == "embedding_grad":
        return [new((case["vocab"], case["cols"]), kind)]
    return [[torch.empty_like(t) for t in state["x"]], new(1, wide)]


def _library():
    """The one handle that the program keeps."""
    global _ops
    if _ops is None:
        from libnd4j_b200.native_ops import NativeOps
        _ops = NativeOps()
    return _ops


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    make = {"layer_norm": _prepare_layer_norm, "layer_norm_grad": _prepare_layer_norm, "log_probs": _prepare_log_probs,
            "log_probs_grad": _prepare_log_probs, "embedding": _prepare_embedding, "embedding_grad": _prepare_embedding,
            "clip": _prepare_clip}[case["op"]]
    state = make(case, gen)
    state["case"] = case
    if own:
        from libnd4j_b200 import shape
        state["ops"] = _library()
        state["out"] = _outputs(case, state)
        state["info"] = {name: shape.shape_info(t.shape) for name, t in state.items() if torch.is_tensor(t) and t.dim() == 2}
        if case["op"].startswith("embedding"):
            state["info"]["out"] = shape.shape_info(state["out"][0].shape)
    return state


# ---- plain forms --------------------------------------------------------------------------------

def _plain_layer_norm(s, case):
    wide = _wide(case["type"])
    x = s["x"].to(wide)
    mean = x.mean(1)
    centred = x - mean[:, None]
    inv = 1 / torch.sqrt((centred * centred).mean(1) + s["epsilon"])
    z = centred * inv[:, None] * s["gain"].to(wide) + s["bias"].to(wide)
    return z.to(s["x"].dtype), mean, inv


def _plain_layer_norm_grad(s, case):
    wide, kind = _wide(case["type"]), s["x"].dtype
    hat = (s["x"].to(wide) - s["mean"][:, None]) * s["invStd"][:, None]
    dz = s["dz"].to(wide)
    d = dz * s["gain"].to(wide)
    dx = (d - d.mean(1, keepdim=True) - hat * (d * hat).mean(1, keepdim=True)) * s["invStd"][:, None]
    return (dx.to(kind), (dz * hat).sum(0, dtype=torch.float64).to(kind), dz.sum(0, dtype=torch.float64).to(kind))


def _plain_log_probs(s, case):
    wide, tokens, k = _wide(case["type"]), s["tokens"], case["k"]
    x = s["logits"].to(wide)
    top = x.amax(1)
    d = (x - top[:, None]) * s["scale"]
    e = torch.exp(d)
    total = e.sum(1)
    log_sum = torch.log(total)
    entropy = log_sum - torch.where(e > 0, d * e, 0).sum(1) / total
    live = tokens >= 0
    chosen = torch.gather(d, 1, tokens.clamp(min=0)[:, None])[:, 0] - log_sum
    zero = torch.zeros_like(top)
    out = [torch.where(live, chosen, zero), torch.where(live, entropy, zero), torch.where(live, top, zero),
           torch.where(live, log_sum, zero)]
    if k:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]      # equal values: lowest index first
        best = torch.gather(d, 1, order) - log_sum[:, None]
        out += [torch.where(live[:, None], order, -1), torch.where(live[:, None], best, 0)]
    return out


def _plain_log_probs_grad(s, case):
    wide, tokens = _wide(case["type"]), s["tokens"]
    log_p = (s["logits"].to(wide) - s["rowMax"][:, None]) * s["scale"] - s["logSum"][:, None]
    p = torch.exp(log_p)
    live = (tokens >= 0).to(wide)[:, None]
    g = s["dLogProbs"][:, None] * live
    d = -g * p
    d.scatter_add_(1, tokens.clamp(min=0)[:, None], g)
    if s["dEntropy"] is not None:
        d -= (s["dEntropy"][:, None] * live) * torch.where(p > 0, p * (log_p + s["entropy"][:, None]), 0)
    return [(d * s["scale"]).to(s["logits"].dtype)]


def _plain_embedding(s, case):
    rows = s["table"][s["tokens"].clamp(min=0)].to(_wide(case["type"])) * s["scale"]
    return [torch.where((s["tokens"] >= 0)[:, None], rows, 0).to(s["table"].dtype)]


def _plain_embedding_grad(s, case):
    total = torch.zeros(case["vocab"] + 1, case["cols"], device="cuda", dtype=torch.float64)
    total.index_add_(0, torch.where(s["tokens"] >= 0, s["tokens"], case["vocab"]), s["dz"].double())
    return [(total[:-1] * s["scale"]).to(s["dz"].dtype)]


def _plain_clip(s, case):
    wide = _wide(case["type"])
    total = sum((t.double() ** 2).sum() for t in s["x"])
    norm = torch.sqrt(total)
    factor = torch.where(norm > s["maxNorm"], s["maxNorm"] / norm, 1.0).to(wide)
    return [(t.to(wide) * factor).to(t.dtype) for t in s["x"]], norm.to(wide)[None]


# ---- the library's calls ------------------------------------------------------------------------

def _own(s, case):
    ops, out, info = s["ops"], s["out"], s["info"]
    dt = {"float": 0, "double": 1, "half": 2}[case["type"]]
    extra = [None, torch.cuda.current_stream().cuda_stream]
    if case["op"] == "layer_norm":
        ops.execLayerNorm(dt, extra, s["x"], info["x"], s["gain"], s["bias"], s["epsilon"], out[0], info["x"], out[1], out[2], [1], 1)
    elif case["op"] == "layer_norm_grad":
        ops.execLayerNormGrad(dt, extra, s["x"], info["x"], s["gain"], s["mean"], s["invStd"], s["dz"], info["dz"],
                              out[0], info["x"], out[1], out[2], [1], 1)
    elif case["op"] == "log_probs":
        best = out[4:] if case["k"] else [None, None]
        ops.execTokenLogProbs(dt, extra, s["logits"], info["logits"], s["tokens"], s["scale"], out[0], out[1], out[2], out[3],
                              case["k"], best[0], best[1])
    elif case["op"] == "log_probs_grad":
        ops.execTokenLogProbsGrad(dt, extra, s["logits"], info["logits"], s["tokens"], s["scale"], s["rowMax"], s["logSum"],
                                  s["entropy"], s["dLogProbs"], s["dEntropy"], out[0], info["logits"])
    elif case["op"] == "embedding":
        ops.execEmbedding(dt, extra, s["table"], info["table"], s["tokens"], s["scale"], out[0], info["out"])
    elif case["op"] == "embedding_grad":
        ops.execEmbeddingGrad(dt, extra, s["tokens"], s["scale"], s["dz"], info["dz"], out[0], info["out"], False)
    else:
        ops.execClipByGlobalNorm(dt, extra, s["x"], out[0], s["lengths"], len(s["lengths"]), s["maxNorm"], out[1])
    return out


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    return {"layer_norm": _plain_layer_norm, "layer_norm_grad": _plain_layer_norm_grad, "log_probs": _plain_log_probs,
            "log_probs_grad": _plain_log_probs_grad, "embedding": _plain_embedding, "embedding_grad": _plain_embedding_grad,
            "clip": _plain_clip}[case["op"]](state, case)


def work(case):
    size, wide = SIZES[case["type"]], 8 if case["type"] == "double" else 4
    op = case["op"]
    if op == "layer_norm":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * size + 2 * case["cols"] * size + 2 * case["rows"] * wide, "flops": 8 * n}
    if op == "layer_norm_grad":
        n = case["rows"] * case["cols"]
        return {"bytes": 3 * n * size + 3 * case["cols"] * size + 2 * case["rows"] * wide, "flops": 14 * n}
    if op == "log_probs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (8 + 4 * wide + case["k"] * (8 + wide)), "flops": 6 * n}
    if op == "log_probs_grad":
        n = case["rows"] * case["vocab"]
        return {"bytes": 2 * n * size + case["rows"] * (8 + 5 * wide), "flops": 8 * n}
    if op == "embedding":
        n = case["tokens"] * case["cols"]
        return {"bytes": 2 * n * size + 8 * case["tokens"], "flops": n}
    if op == "embedding_grad":
        n, table = case["tokens"] * case["cols"], case["vocab"] * case["cols"]
        return {"bytes": (n + table) * size + 8 * case["tokens"], "flops": n + table}
    n = case["total"]
    return {"bytes": 2 * n * size + wide, "flops": 3 * n}


# ---- the operators' definitions in 64 bits ------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "layer_norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0)
        inv = (var + s["epsilon"]).pow(-0.5)
        z = torch.addcmul(s["bias"].double(), (x - mean.unsqueeze(1)) * s["gain"].double(), inv.unsqueeze(1))
        return z, mean, inv
    if op == "layer_norm_grad":
        n = case["cols"]
        inv = s["invStd"].double().unsqueeze(1)
        hat = s["x"].double().sub_(s["mean"].double().unsqueeze(1)).mul_(inv)
        dz = s["dz"].double()
        d_gain, d_bias = torch.einsum("ij,ij->j", dz, hat), dz.sum(0)
        dz *= s["gain"].double()
        a, b = dz.sum(1, keepdim=True), torch.einsum("ij,ij->i", dz, hat).unsqueeze(1)
        return inv / n * (n * dz - a - hat * b), d_gain, d_bias
    if op == "log_probs":
        y = s["logits"].double() * s["scale"]
        log_p = y - torch.logsumexp(y, dim=1, keepdim=True)
        entropy = -(log_p.exp() * log_p.clamp(min=-1e6)).sum(1)
        top = s["logits"].double().max(1).values
        out = [log_p.gather(1, s["tokens"].clamp(min=0).unsqueeze(1)).squeeze(1), entropy, top,
               torch.logsumexp(y, dim=1) - top * s["scale"]]
        if case["k"]:
            best, ids = _best(s["logits"], case["k"])
            out += [ids, log_p.gather(1, ids)]
        for t, pad in zip(out, [0, 0, 0, 0, -1, 0]):
            t[s["tokens"] < 0] = pad
        return out
    if op == "log_probs_grad":
        y = s["logits"].double().mul_(s["scale"])
        y -= (s["rowMax"].double() * s["scale"] + s["logSum"].double()).unsqueeze(1)
        p = y.exp()
        d = p * -s["dLogProbs"].double().unsqueeze(1)
        rows = torch.arange(case["rows"], device="cuda")
        d[rows, s["tokens"].clamp(min=0)] += s["dLogProbs"].double()
        if s["dEntropy"] is not None:
            y.clamp_(min=-1e6).add_(s["entropy"].double().unsqueeze(1))
            d -= p * y * s["dEntropy"].double().unsqueeze(1)
        d *= s["scale"]
        d[s["tokens"] < 0] = 0
        return [d]
    if op == "embedding":
        live = (s["tokens"] >= 0).double().unsqueeze(1)
        return [torch.index_select(s["table"], 0, s["tokens"].clamp(min=0)).double() * (live * s["scale"])]
    if op == "embedding_grad":
        order = torch.argsort(s["tokens"], stable=True)[int((s["tokens"] < 0).sum()):]
        ids, counts = torch.unique_consecutive(s["tokens"][order], return_counts=True)
        grad = torch.zeros(case["vocab"], case["cols"], device="cuda", dtype=torch.float64)
        grad[ids] = torch.segment_reduce(s["dz"].double()[order], "sum", lengths=counts, axis=0) * s["scale"]
        return [grad]
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(t, dtype=torch.float64) for t in s["x"]]))
    factor = min(1.0, s["maxNorm"] / float(norm))
    return [t.double() * factor for t in s["x"]], norm[None]


def _best(logits, k):
    """The k largest of each row and where they stand, equal values in the order of their indices."""
    rest = logits.double().clone()
    ids = []
    at = torch.arange(rest.shape[1], device="cuda")
    for _ in range(k):
        top = rest.max(1, keepdim=True).values
        ids.append(torch.where(rest == top, at, rest.shape[1]).min(1).values)
        rest.scatter_(1, ids[-1].unsqueeze(1), -math.inf)
    ids = torch.stack(ids, 1)
    return logits.double().gather(1, ids), ids
