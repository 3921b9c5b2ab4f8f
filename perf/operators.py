"""The training-side operators at the two ends of a decoder, in plain torch and as the calls of this library.

Three operators, each with its gradient:

* ``lce``      softmax cross entropy of ``x W^T + b`` over a large vocabulary, without keeping the logits
* ``embed``    embedding lookup with a scale, and the gradient of the table
* ``distill``  distillation from the top logits of a teacher

The plain forms spell the formulas out with elementary operations in 32 bits and round once at the end; ``exact``
has the same results from the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ---------------------------------------------------------------------------------------------------


def listed():
    return [
        # the loss of the tiny decoder (vocab 256, d 64, 4 x 32 tokens): a call that costs little more than its launches
        dict(name="lce tiny step", op="lce", tokens=128, vocab=256, dim=64, dtype="bf16", bias=True, train=True),
        # the same kind of model in fp32, where the framework promises fp32 products; sizes off every tile
        dict(name="lce fp32 step", op="lce", tokens=301, vocab=1003, dim=97, dtype="f32", bias=True, train=True),
        # evaluation (perplexity) of the 2B-class decoder on two sequences: no gradient
        dict(name="lce 2B-class eval", op="lce", tokens=4096, vocab=32000, dim=2048, dtype="bf16", bias=False, train=False),
        # a ragged fine-tuning batch: odd token count and vocabulary, prompt tokens left out of the loss
        dict(name="lce ragged step", op="lce", tokens=1543, vocab=50021, dim=1000, dtype="bf16", bias=True, train=True),
        # a training step's loss of the 2B-class decoder: 8 sequences of 2048
        dict(name="lce 2B-class step", op="lce", tokens=16384, vocab=32000, dim=2048, dtype="bf16", bias=False, train=True),
        # the tiny decoder's lookup and gradient
        dict(name="embed tiny step", op="embed", tokens=128, vocab=256, dim=64, dtype="f32", grad="f32", skew=False),
        # odd sizes, natural token frequencies (a few tokens make up most of the text), a large table
        dict(name="embed ragged step", op="embed", tokens=10007, vocab=128001, dim=1001, dtype="bf16", grad="f32", skew=True),
        # the 2B-class decoder: 32 x 2048 tokens, fp32 table and gradient
        dict(name="embed 2B-class step", op="embed", tokens=65536, vocab=32000, dim=2048, dtype="f32", grad="f32", skew=True),
        # the tiny decoder as a student
        dict(name="distill tiny step", op="distill", rows=128, vocab=256, k=8, dtype="f32", tau=1.0),
        # a handful of positions over a large vocabulary: one row has to be spread over the GPU
        dict(name="distill few rows", op="distill", rows=5, vocab=200003, k=50, dtype="f32", tau=2.0),
        # bf16 logits with an odd row length
        dict(name="distill ragged step", op="distill", rows=2047, vocab=128001, k=20, dtype="bf16", tau=1.0),
        # the 2B-class decoder's logits of 4 sequences of 2048
        dict(name="distill 2B-class step", op="distill", rows=8192, vocab=32000, k=64, dtype="f32", tau=2.0),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["lce", "embed", "distill"])
    if op == "lce":
        if rng.random() < 0.2:  # the fp32 route runs at the sizes of small models
            return dict(op=op, tokens=_log_uniform(rng, 1, 1024), vocab=_log_uniform(rng, 64, 4096), dim=_log_uniform(rng, 16, 512),
                        dtype="f32", bias=rng.random() < 0.5, train=rng.random() < 0.7)
        dim = 8 * _log_uniform(rng, 8, 256) if rng.random() < 0.85 else _log_uniform(rng, 16, 300)
        small = dim % 8 != 0
        return dict(op=op, tokens=_log_uniform(rng, 1, 512 if small else 12288), vocab=_log_uniform(rng, 128, 2048 if small else 40000),
                    dim=dim, dtype="bf16", bias=rng.random() < 0.5, train=rng.random() < 0.7)
    if op == "embed":
        return dict(op=op, tokens=_log_uniform(rng, 1, 60000), vocab=_log_uniform(rng, 64, 130000), dim=_log_uniform(rng, 32, 2048),
                    dtype=rng.choice(["bf16", "f32"]), grad=rng.choice(["bf16", "f32"]), skew=rng.random() < 0.6)
    vocab = _log_uniform(rng, 64, 200000)
    return dict(op=op, rows=_log_uniform(rng, 1, max(2, min(8192, 262144000 // vocab))), vocab=vocab, k=min(vocab, _log_uniform(rng, 1, 128)),
                dtype=rng.choice(["bf16", "f32"]), tau=rng.choice([1.0, 1.5, 2.0, 4.0]))


# ---- inputs --------------------------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, sigma=1.0):
        return torch.randn(*shape, generator=gen, device="cuda") * sigma

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    t = DTYPES[case["dtype"]]
    if case["op"] == "lce":
        tokens, vocab, dim = case["tokens"], case["vocab"], case["dim"]
        # a normalised hidden state and an output matrix that gives logits of a few units; every sixteenth row or so is a prompt token
        labels = torch.floor(uniform(tokens) * vocab).clamp_(max=vocab - 1)
        labels = torch.where(uniform(tokens) < 0.06, torch.full_like(labels, -1.0), labels)
        labels[0] = vocab // 2
        return dict(case, x=normal(tokens, dim).to(t), w=normal(vocab, dim, sigma=2.0 / math.sqrt(dim)).to(t),
                    b=normal(vocab, sigma=0.2) if case["bias"] else None, labels=labels)
    if case["op"] == "embed":
        tokens, vocab, dim = case["tokens"], case["vocab"], case["dim"]
        u = uniform(tokens)
        # token frequencies that fall with the rank, or uniform ids
        ids = torch.floor(torch.exp(u * math.log(vocab + 1.0))) - 1.0 if case["skew"] else torch.floor(u * vocab)
        return dict(case, ids=ids.clamp_(0, vocab - 1), table=normal(vocab, dim, sigma=0.02).to(t), dout=normal(tokens, dim).to(t),
                    scale=math.sqrt(dim))
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    logits = normal(rows, vocab, sigma=2.5)
    top = torch.topk(logits + normal(rows, vocab, sigma=0.7), k, dim=1)
    ids = top.indices.float()
    # a teacher that stops early lists fewer entries: the rest are marked -1
    short = uniform(rows, k) < 0.05
    short[:, 0] = False
    return dict(case, logits=logits.to(t), ids=torch.where(short, torch.full_like(ids, -1.0), ids), teacher=top.values.contiguous(),
                weight=0.5 + uniform(rows))


# ---- one pass ------------------------------------------------------------------------------------------------


def _plain_lce(s):
    t = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"]
    counted = s["labels"] >= 0
    label = s["labels"].clamp(min=0).long()
    top = z.max(dim=1).values
    lse = top + torch.log(torch.exp(z - top[:, None]).sum(dim=1))
    at = z.gather(1, label[:, None])[:, 0]
    loss = torch.where(counted, lse - at, torch.zeros_like(lse))
    out = {"loss": loss, "lse": lse, "summary": torch.stack([loss.sum(), counted.sum().float(), 1.0 / counted.sum().float()])}
    if s["train"]:
        g = torch.where(counted, 1.0 / counted.sum().float(), torch.zeros_like(lse))
        dz = torch.exp(z - lse[:, None])
        rows = torch.arange(dz.shape[0], device=dz.device)
        dz[rows, label] -= 1.0
        dz *= g[:, None]
        out["dx"] = (dz @ w).to(t)
        out["dw"] = (dz.t() @ x).to(t)
        if s["b"] is not None:
            out["db"] = dz.sum(dim=0)
    return out


def _plain_embed(s):
    at = s["ids"].long()
    out = (s["table"][at].float() * s["scale"]).to(s["table"].dtype)
    grad = torch.zeros(s["vocab"], s["dim"], device=at.device)
    grad.index_add_(0, at, s["dout"].float())
    return {"out": out, "dtable": (grad * s["scale"]).to(DTYPES[s["grad"]])}


def _plain_distill(s):
    tau = s["tau"]
    z = s["logits"].float() / tau
    top = z.max(dim=1).values
    lse = top + torch.log(torch.exp(z - top[:, None]).sum(dim=1))
    there = s["ids"] >= 0
    at = s["ids"].clamp(min=0).long()
    teacher = torch.where(there, s["teacher"] / tau, torch.full_like(s["teacher"], -math.inf))
    teacher = teacher - teacher.max(dim=1, keepdim=True).values
    q = torch.exp(teacher)
    total = q.sum(dim=1, keepdim=True)
    q = q / total
    gap = teacher - torch.log(total) - (z.gather(1, at) - lse[:, None])
    loss = tau * tau * torch.where(there, q * gap, torch.zeros_like(q)).sum(dim=1)
    dz = torch.exp(z - lse[:, None])
    dz.scatter_add_(1, at, -q)
    dz *= (tau * s["weight"])[:, None]
    return {"loss": loss, "lse": lse, "dlogits": dz.to(s["logits"].dtype)}


def _code(bfb, t):
    return bfb.F32 if t == torch.float32 else bfb.BF16


def _workspace(bfb, query, *args):
    import ctypes
    n = ctypes.c_size_t(0)
    bfb.check(query(*args, ctypes.byref(n)))
    return torch.empty(max(1, n.value), dtype=torch.uint8, device="cuda"), n.value


def _own_lce(s, bfb, lib, stream):
    tokens, vocab, dim, train = s["tokens"], s["vocab"], s["dim"], s["train"]
    x, w, b = s["x"], s["w"], s["b"]
    code = _code(bfb, x.dtype)
    if "kept" not in s:  # what a training loop allocates once
        ws, size = _workspace(bfb, lib.bfb_linear_cross_entropy_workspace, code, tokens, vocab, dim, int(train))
        s["kept"] = dict(ws=ws, size=size, loss=x.new_empty(tokens, dtype=torch.float32), lse=x.new_empty(tokens, dtype=torch.float32),
                         summary=x.new_empty(3, dtype=torch.float32), dx=torch.empty_like(x) if train else None,
                         dw=torch.empty_like(w) if train else None, db=torch.empty_like(b) if train and b is not None else None)
    k = s["kept"]
    bias = None if b is None else b.data_ptr()
    summary = k["summary"].data_ptr()
    bfb.check(lib.bfb_linear_cross_entropy_fwd(
        x.data_ptr(), dim, w.data_ptr(), dim, bias, s["labels"].data_ptr(), k["loss"].data_ptr(), k["lse"].data_ptr(), summary, code,
        tokens, vocab, dim, None, k["ws"].data_ptr(), k["size"], None, stream))
    out = {"loss": k["loss"], "lse": k["lse"], "summary": k["summary"]}
    if train:
        # the mean over the counted rows: its scale is the third word of the forward's summary
        bfb.check(lib.bfb_linear_cross_entropy_bwd(
            x.data_ptr(), dim, w.data_ptr(), dim, bias, s["labels"].data_ptr(), k["lse"].data_ptr(), None, summary + 8, 1.0,
            k["dx"].data_ptr(), dim, k["dw"].data_ptr(), dim, None if b is None else k["db"].data_ptr(), code, code,
            tokens, vocab, dim, k["ws"].data_ptr(), k["size"], None, stream))
        out["dx"], out["dw"] = k["dx"], k["dw"]
        if b is not None:
            out["db"] = k["db"]
    return out


def _own_embed(s, bfb, lib, stream):
    tokens, vocab, dim = s["tokens"], s["vocab"], s["dim"]
    if "kept" not in s:
        ws, size = _workspace(bfb, lib.bfb_embed_scaled_bwd_workspace, tokens, vocab, dim)
        s["kept"] = dict(ws=ws, size=size, out=torch.empty_like(s["dout"]),
                         dtable=s["table"].new_empty(vocab, dim, dtype=DTYPES[s["grad"]]))
    k = s["kept"]
    code = _code(bfb, s["table"].dtype)
    bfb.check(lib.bfb_embed_scaled(s["ids"].data_ptr(), s["table"].data_ptr(), code, k["out"].data_ptr(), code, dim, tokens, vocab, dim,
                                   s["scale"], None, stream))
    bfb.check(lib.bfb_embed_scaled_bwd(s["ids"].data_ptr(), s["dout"].data_ptr(), code, dim, k["dtable"].data_ptr(),
                                       _code(bfb, k["dtable"].dtype), tokens, vocab, dim, s["scale"], 0, k["ws"].data_ptr(), k["size"],
                                       stream))
    return {"out": k["out"], "dtable": k["dtable"]}


def _own_distill(s, bfb, lib, stream):
    rows, vocab, count = s["rows"], s["vocab"], s["k"]
    z = s["logits"]
    if "kept" not in s:
        s["kept"] = dict(loss=z.new_empty(rows, dtype=torch.float32), lse=z.new_empty(rows, dtype=torch.float32), dz=torch.empty_like(z))
    k = s["kept"]
    code = _code(bfb, z.dtype)
    bfb.check(lib.bfb_distill_topk(z.data_ptr(), code, vocab, s["ids"].data_ptr(), s["teacher"].data_ptr(), bfb.F32, count, s["tau"],
                                   s["weight"].data_ptr(), None, 1.0, k["loss"].data_ptr(), k["lse"].data_ptr(), k["dz"].data_ptr(), code,
                                   vocab, rows, vocab, None, stream))
    return {"loss": k["loss"], "lse": k["lse"], "dlogits": k["dz"]}


def run(state):
    if own:
        import blackforge_b200 as bfb
        form = {"lce": _own_lce, "embed": _own_embed, "distill": _own_distill}[state["op"]]
        return form(state, bfb, bfb.lib(), torch.cuda.current_stream().cuda_stream)
    return {"lce": _plain_lce, "embed": _plain_embed, "distill": _plain_distill}[state["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "lce":
        tokens, vocab, dim = case["tokens"], case["vocab"], case["dim"]
        operands = (tokens + vocab) * dim * e + (vocab * 4 if case["bias"] else 0)
        total = operands + tokens * 12
        if case["train"]:
            total += operands
        return {"bytes": total, "flops": (6 if case["train"] else 2) * tokens * vocab * dim}
    if case["op"] == "embed":
        tokens, vocab, dim = case["tokens"], case["vocab"], case["dim"]
        g = 4 if case["grad"] == "f32" else 2
        rows = min(tokens, vocab)
        return {"bytes": tokens * 4 + rows * dim * e + 2 * tokens * dim * e + vocab * dim * g, "flops": 2 * tokens * dim}
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    return {"bytes": 2 * rows * vocab * e + rows * k * 8 + rows * 12, "flops": 6 * rows * vocab}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lce":
        x = s["x"].double().requires_grad_(case["train"])
        w = s["w"].double().requires_grad_(case["train"])
        b = None if s["b"] is None else s["b"].double().requires_grad_(case["train"])
        z = torch.nn.functional.linear(x, w, b)
        label = s["labels"].long()
        loss = torch.nn.functional.cross_entropy(z, label, ignore_index=-1, reduction="none")
        count = (label != -1).sum().double()
        out = {"loss": loss.detach(), "lse": torch.logsumexp(z.detach(), 1), "summary": torch.stack([loss.detach().sum(), count, 1 / count])}
        if case["train"]:
            (loss.sum() / count).backward()
            out["dx"], out["dw"] = x.grad, w.grad
            if b is not None:
                out["db"] = b.grad
        return out
    if case["op"] == "embed":
        order = torch.argsort(s["ids"], stable=True)
        seen, counts = torch.unique_consecutive(s["ids"][order].long(), return_counts=True)
        grad = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda")
        width = 128
        for c in range(0, case["dim"], width):  # sums over each token's run, a few columns at a time
            grad[seen, c:c + width] = torch.segment_reduce(s["dout"][:, c:c + width].double()[order], "sum", lengths=counts, axis=0)
        return {"out": torch.nn.functional.embedding(s["ids"].long(), s["table"].double()) * s["scale"], "dtable": grad * s["scale"]}
    z = s["logits"].double().requires_grad_()
    there = s["ids"] >= 0
    log_p = torch.log_softmax(z / case["tau"], dim=1).gather(1, s["ids"].clamp(min=0).long())
    teacher = (s["teacher"].double() / case["tau"]).masked_fill(~there, -math.inf)
    log_q = torch.log_softmax(teacher, dim=1)
    part = log_q.exp() * (log_q.masked_fill(~there, 0.0) - log_p)
    loss = case["tau"] ** 2 * part.masked_fill(~there, 0.0).sum(1)
    (loss * s["weight"].double()).sum().backward()
    return {"loss": loss.detach(), "lse": torch.logsumexp(z.detach() / case["tau"], 1), "dlogits": z.grad}
