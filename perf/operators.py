"""What the vocabulary operators are measured on: embedding lookup, vocabulary loss and distillation loss.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``prepare()`` makes a case's inputs on the GPU
and ``run()`` computes one pass: in elementary torch operations in 32 bits where ``own`` is false, through
``HIPDriver``'s entry points where it is true.  ``exact()`` computes the same outputs in 64 bits from the definitions:

  embedding   out[t] = scale * table[ids[t]] (zero for the padding id); dtable[v] = scale * sum of dout[t] over ids[t] == v
  vocab loss  l = x w^T + bias, loss[t] = log sum exp l[t] - l[t][label[t]] (zero for an ignored label);
              G[t][v] = loss_grad[t] * (softmax(l[t])[v] - [v == label[t]]), dx = G w, dw = G^T x, db = column sums of G
  distill     q = softmax(top_logits / T) over a token's valid entries, p = softmax(logits / T) over the vocabulary,
              loss[t] = T^2 * sum q (log q - log p[top_ids]), dlogits[t] = loss_grad[t] * T * (p - q scattered to top_ids)
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
IGNORED = -1          # padding id, ignored label, absent entry of a top list


def listed():
    return [
        # one decoding step of eight sequences: a launch's latency
        {"name": "embedding_step", "op": "embedding", "pass": "forward", "dtype": "bf16", "tokens": 8, "width": 4096,
         "vocab": 32000},
        # the lookup of a long training batch
        {"name": "embedding_batch", "op": "embedding", "pass": "forward", "dtype": "bf16", "tokens": 65536,
         "width": 2048, "vocab": 131072},
        # gradient of a small table with a width that is no multiple of a vector load, in full precision
        {"name": "embedding_grad_odd", "op": "embedding", "pass": "backward", "dtype": "f32", "tokens": 4099,
         "width": 1001, "vocab": 10007},
        # gradient of the largest table, most tokens on few ids as text has them
        {"name": "embedding_grad_large", "op": "embedding", "pass": "backward", "dtype": "bf16", "tokens": 65536,
         "width": 4096, "vocab": 131072},
        # scoring the candidates of a few sequences: bound by reading the weights
        {"name": "vocab_score", "op": "vocab", "pass": "forward", "dtype": "bf16", "tokens": 16, "width": 1024,
         "vocab": 32000, "bias": False},
        # evaluating perplexity on a batch
        {"name": "vocab_eval", "op": "vocab", "pass": "forward", "dtype": "bf16", "tokens": 4096, "width": 2048,
         "vocab": 131072, "bias": False},
        # a training step of a classifier head in the framework's own type, with a bias (1000 classes, 4096 wide)
        {"name": "vocab_train_classes", "op": "vocab", "pass": "train", "dtype": "f32", "tokens": 256, "width": 4096,
         "vocab": 1000, "bias": True},
        # a training step in full precision over a middling vocabulary
        {"name": "vocab_train_f32", "op": "vocab", "pass": "train", "dtype": "f32", "tokens": 2048, "width": 1024,
         "vocab": 32768, "bias": False},
        # ragged sizes: a packed batch with an odd number of tokens, odd vocabulary, width not a whole number of tiles
        {"name": "vocab_train_ragged", "op": "vocab", "pass": "train", "dtype": "bf16", "tokens": 1023, "width": 1000,
         "vocab": 50021, "bias": True},
        # the largest training step
        {"name": "vocab_train_large", "op": "vocab", "pass": "train", "dtype": "bf16", "tokens": 8192, "width": 4096,
         "vocab": 131072, "bias": False},
        # distilling the 1000-class layer of a small batch
        {"name": "distill_classes", "op": "distill", "pass": "train", "dtype": "f32", "tokens": 32, "vocab": 1000,
         "top": 10},
        # distilling a language model's batch
        {"name": "distill_large", "op": "distill", "pass": "train", "dtype": "bf16", "tokens": 4096, "vocab": 131072,
         "top": 64},
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of [low, high], a multiple of 64 half of the time."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and n >= 128:
        n = n // 64 * 64
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["embedding", "vocab", "distill"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "embedding":
        return {"op": op, "pass": rng.choice(["forward", "backward"]), "dtype": dtype, "tokens": _spread(rng, 1, 65536),
                "width": _spread(rng, 32, 4096), "vocab": _spread(rng, 500, 65536 if dtype == "f32" else 131072)}
    if op == "distill":
        return {"op": op, "pass": rng.choice(["forward", "train"]), "dtype": dtype,
                "tokens": _spread(rng, 1, 2048 if dtype == "f32" else 4096), "vocab": _spread(rng, 500, 131072),
                "top": _spread(rng, 1, 128)}
    # the widest and longest cases in full precision stop at a sixteenth of the largest listed one's products
    f32 = dtype == "f32"
    return {"op": op, "pass": rng.choice(["forward", "train"]), "dtype": dtype,
            "tokens": _spread(rng, 1, 2048 if f32 else 8192), "width": _spread(rng, 64, 2048 if f32 else 4096),
            "vocab": _spread(rng, 500, 65536 if f32 else 131072), "bias": rng.random() < 0.5}


def _text_ids(count, vocab, gen):
    """Ids as text has them: the frequency of the r-th commonest falls as 1 / (r + 2), over a shuffled vocabulary."""
    weight = 1.0 / (torch.arange(vocab, device="cuda", dtype=torch.float64) + 2.0)
    at = torch.cumsum(weight, 0)
    u = torch.rand(count, generator=gen, device="cuda", dtype=torch.float64) * at[-1]
    rank = torch.searchsorted(at, u).clamp_(max=vocab - 1)
    return torch.randperm(vocab, generator=gen, device="cuda")[rank].to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    t, v, dtype = case["tokens"], case["vocab"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    s = {"case": dict(case)}
    if case["op"] == "embedding":
        w = case["width"]
        s["scale"] = math.sqrt(w)
        ids = _text_ids(t, v, gen)
        pad = torch.rand(t, generator=gen, device="cuda") < 0.02
        pad[0] = False
        s["ids"] = torch.where(pad, torch.full_like(ids, IGNORED), ids)
        if case["pass"] == "forward":
            s["table"] = (normal(v, w) / math.sqrt(w)).to(dtype)
        else:
            s["dout"] = (normal(t, w) * 1e-3).to(dtype)
    elif case["op"] == "vocab":
        w = case["width"]
        weights = normal(v, w) / math.sqrt(w)
        labels = _text_ids(t, v, gen)
        # hidden states of a model that has learned something: they lean towards the label's row
        x = normal(t, w) * 2.0 + weights[labels.long()] * (3.0 * torch.rand(t, 1, generator=gen, device="cuda"))
        ignored = torch.rand(t, generator=gen, device="cuda") < 0.05
        ignored[0] = False
        s["labels"] = torch.where(ignored, torch.full_like(labels, IGNORED), labels)
        s["x"], s["w"] = x.to(dtype), weights.to(dtype)
        s["bias"] = normal(v).to(dtype) if case["bias"] else None
        kept = (~ignored).sum().clamp(min=1)
        s["loss_grad"] = torch.full((t,), 1.0, device="cuda") / kept        # the mean over the tokens that count
    else:
        k = min(case["top"], v)
        s["temperature"] = 2.0
        teacher = normal(t, v) * 2.0
        # the student leans towards its teacher
        s["logits"] = (0.7 * teacher + normal(t, v)).to(dtype)
        top, at = torch.topk(teacher, k, dim=1)
        absent = torch.rand(t, generator=gen, device="cuda") < 0.1          # rows whose list is shorter
        length = torch.where(absent, torch.full((t,), max(1, k // 2), device="cuda"), torch.full((t,), k, device="cuda"))
        valid = torch.arange(k, device="cuda")[None, :] < length[:, None]
        s["top_ids"] = torch.where(valid, at, torch.full_like(at, IGNORED)).to(torch.int32).contiguous()
        s["top_logits"] = torch.where(valid, top, torch.zeros_like(top)).contiguous()
        s["loss_grad"] = torch.full((t,), 1.0 / t, device="cuda")
    if own:
        _prepare_own(s)
    return s


def _prepare_own(s):
    """The handle, argument block, outputs and workspace that a program keeps from call to call."""
    from caffecontroll_amd import HIPDriver
    from caffecontroll_amd.driver import BF16, F32, distill_loss_args, embedding_args, vocab_loss_args
    case = s["case"]
    drv = s["drv"] = HIPDriver(torch.cuda.current_device())
    drv.set_stream(torch.cuda.current_stream().cuda_stream)
    dtype = BF16 if case["dtype"] == "bf16" else F32
    t, v = case["tokens"], case["vocab"]
    if case["op"] == "embedding":
        s["args"] = embedding_args(t, case["width"], v, dtype, scale=s["scale"], padding_id=IGNORED)
        s["bytes"] = drv.embedding_workspace_bytes(s["args"]) if case["pass"] == "backward" else 0
        rows = v if case["pass"] == "backward" else t
        s["out"] = torch.empty((rows, case["width"]), dtype=TYPES[case["dtype"]], device="cuda")
    else:
        s["loss"], s["lse"] = torch.empty(t, device="cuda"), torch.empty(t, device="cuda")
        if case["op"] == "vocab":
            s["args"] = vocab_loss_args(t, case["width"], v, dtype, ignore_label=IGNORED)
            s["bytes"] = drv.vocab_loss_workspace_bytes(s["args"])
            if case["pass"] == "train":
                s["dx"], s["dw"] = torch.empty_like(s["x"]), torch.empty_like(s["w"])
                s["db"] = torch.empty_like(s["bias"]) if case["bias"] else None
        else:
            s["args"] = distill_loss_args(t, v, s["top_ids"].shape[1], dtype, temperature=s["temperature"])
            s["bytes"] = drv.distill_loss_workspace_bytes(s["args"])
            if case["pass"] == "train":
                s["dlogits"] = torch.empty_like(s["logits"])
    s["workspace"] = torch.empty(max(16, s["bytes"]), dtype=torch.uint8, device="cuda")


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    case, drv, a, ws, n = s["case"], s["drv"], s["args"], s["workspace"], s["bytes"]
    if case["op"] == "embedding":
        if case["pass"] == "forward":
            drv.embedding_forward(s["out"], s["table"], s["ids"], a)
        else:
            drv.embedding_backward(s["out"], s["dout"], s["ids"], a, ws, n)
        return s["out"]
    if case["op"] == "vocab":
        if case["pass"] == "forward":
            drv.vocab_loss_forward(s["loss"], s["lse"], s["x"], s["w"], s["bias"], s["labels"], a, ws, n)
            return s["loss"], s["lse"]
        drv.vocab_loss_forward_backward(s["loss"], s["lse"], s["dx"], s["dw"], s["db"], s["x"], s["w"], s["bias"],
                                        s["labels"], s["loss_grad"], a, ws, n)
        return [x for x in (s["loss"], s["lse"], s["dx"], s["dw"], s["db"]) if x is not None]
    if case["pass"] == "forward":
        drv.distill_loss_forward(s["loss"], s["lse"], s["logits"], s["top_ids"], s["top_logits"], a, ws, n)
        return s["loss"], s["lse"]
    drv.distill_loss_forward_backward(s["loss"], s["lse"], s["dlogits"], s["logits"], s["top_ids"], s["top_logits"],
                                      s["loss_grad"], a, ws, n)
    return s["loss"], s["lse"], s["dlogits"]


def _run_plain(s):
    case = s["case"]
    dtype = TYPES[case["dtype"]]
    if case["op"] == "embedding":
        ids = s["ids"].long()
        keep = ids >= 0
        if case["pass"] == "forward":
            rows = s["table"][ids.clamp(min=0)].float()
            return torch.where(keep[:, None], rows * s["scale"], torch.zeros((), device="cuda")).to(dtype)
        # padding tokens add to one row more, which is left off
        grad = torch.zeros((case["vocab"] + 1, case["width"]), device="cuda")
        grad.index_add_(0, torch.where(keep, ids, torch.full_like(ids, case["vocab"])), s["dout"].float())
        return (grad[:-1] * s["scale"]).to(dtype)
    if case["op"] == "vocab":
        x, w = s["x"].float(), s["w"].float()
        labels = s["labels"].long()
        keep = labels >= 0
        at = labels.clamp(min=0)[:, None]
        logits = x @ w.t()
        if s["bias"] is not None:
            logits = logits + s["bias"].float()
        top = logits.amax(1, keepdim=True)
        e = torch.exp(logits - top)
        total = e.sum(1, keepdim=True)
        lse = (top + torch.log(total))[:, 0]
        loss = torch.where(keep, lse - logits.gather(1, at)[:, 0], torch.zeros_like(lse))
        if case["pass"] == "forward":
            return loss, lse
        g = e / total
        g.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
        g = g * torch.where(keep, s["loss_grad"], torch.zeros_like(lse))[:, None]
        grads = [(g @ w).to(dtype), (g.t() @ x).to(dtype)]
        if s["bias"] is not None:
            grads.append(g.sum(0).to(dtype))
        return [loss, lse] + grads
    t = s["temperature"]
    z = s["logits"].float() / t
    ids = s["top_ids"].long()
    valid = ids >= 0
    at = ids.clamp(min=0)
    teacher = torch.where(valid, s["top_logits"] / t, torch.full((), -float("inf"), device="cuda"))
    logq = teacher - teacher.amax(1, keepdim=True)
    logq = logq - torch.log(torch.exp(logq).sum(1, keepdim=True))
    q = torch.exp(logq)
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    term = q * (logq - (z.gather(1, at) - lse))
    loss = t * t * torch.where(valid, term, torch.zeros_like(term)).sum(1)
    if case["pass"] == "forward":
        return loss, lse[:, 0]
    g = (e / total).scatter_add_(1, at, -q)
    return loss, lse[:, 0], (g * (s["loss_grad"] * t)[:, None]).to(dtype)


def work(case):
    t, v, b = case["tokens"], case["vocab"], SIZE[case["dtype"]]
    if case["op"] == "embedding":
        row = case["width"] * b
        if case["pass"] == "forward":
            return {"bytes": t * 4 + 2 * t * row, "flops": t * case["width"]}
        return {"bytes": t * 4 + (t + v) * row, "flops": t * case["width"]}
    if case["op"] == "vocab":
        w = case["width"]
        bias = v * b if case["bias"] else 0
        if case["pass"] == "forward":
            return {"bytes": (t + v) * w * b + bias + t * 12, "flops": 2 * t * w * v}
        return {"bytes": 2 * (t + v) * w * b + 2 * bias + t * 16, "flops": 6 * t * w * v}
    lists = t * min(case["top"], v) * 8 + t * 12
    passes = 1 if case["pass"] == "forward" else 2
    return {"bytes": passes * t * v * b + lists, "flops": (3 if passes == 1 else 6) * t * v}


def exact(case, seed):
    """The same outputs from the definitions in 64 bits, a slice of the tokens (or of the vocabulary) at a time."""
    s = prepare(case, seed)
    t, v = case["tokens"], case["vocab"]
    f64 = torch.float64
    if case["op"] == "embedding":
        ids = s["ids"].long()
        if case["pass"] == "forward":
            out = torch.zeros((t, case["width"]), dtype=f64, device="cuda")
            at = torch.nonzero(ids >= 0)[:, 0]
            out[at] = s["table"].index_select(0, ids[at]).to(f64) * s["scale"]
            return out
        # prefix sums over the tokens in the order of their ids: a row's gradient is a difference of two of them
        order = torch.argsort(ids, stable=True)
        begin = torch.searchsorted(ids[order], torch.arange(v + 1, device="cuda"))
        out = torch.empty((v, case["width"]), dtype=f64, device="cuda")
        for c in range(0, case["width"], 256):
            part = s["dout"][:, c:c + 256].to(f64)[order]
            sums = torch.zeros((t + 1, part.shape[1]), dtype=f64, device="cuda")
            torch.cumsum(part, 0, out=sums[1:])
            out[:, c:c + 256] = (sums[begin[1:]] - sums[begin[:-1]]) * s["scale"]
        return out
    if case["op"] == "vocab":
        x, w = s["x"].to(f64), s["w"].to(f64)
        bias = torch.zeros(v, dtype=f64, device="cuda") if s["bias"] is None else s["bias"].to(f64)
        loss, lse = torch.zeros(t, dtype=f64, device="cuda"), torch.zeros(t, dtype=f64, device="cuda")
        train = case["pass"] == "train"
        if train:
            dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias)
        for r in range(0, t, 1024):
            rows = torch.arange(r, min(t, r + 1024), device="cuda")
            logits = torch.addmm(bias, x[rows], w.t())
            lse[rows] = torch.logsumexp(logits, 1)
            here = torch.nonzero(s["labels"][rows] >= 0)[:, 0]
            at = s["labels"][rows][here].long()
            loss[rows[here]] = lse[rows[here]] - logits[here, at]
            if train:
                weight = torch.zeros(len(rows), dtype=f64, device="cuda")
                weight[here] = s["loss_grad"][rows[here]].to(f64)
                g = torch.exp(logits - lse[rows][:, None])
                g[here, at] -= 1.0
                g *= weight[:, None]
                dx[rows] = g @ w
                dw.addmm_(g.t(), x[rows])
                db += g.sum(0)
        if not train:
            return loss, lse
        return [loss, lse, dx, dw] + ([db] if s["bias"] is not None else [])
    temp = s["temperature"]
    loss, lse = torch.zeros(t, dtype=f64, device="cuda"), torch.zeros(t, dtype=f64, device="cuda")
    grad = torch.zeros((t, v), dtype=f64, device="cuda") if case["pass"] == "train" else None
    for r in range(0, t, 1024):
        rows = slice(r, min(t, r + 1024))
        logp = torch.log_softmax(s["logits"][rows].to(f64) / temp, 1)
        lse[rows] = s["logits"][rows, 0].to(f64) / temp - logp[:, 0]
        ids = s["top_ids"][rows].long()
        teacher = (s["top_logits"][rows].to(f64) / temp).masked_fill(ids < 0, -float("inf"))
        logq = torch.log_softmax(teacher, 1)
        q = torch.exp(logq)
        inner = q * (logq.masked_fill(ids < 0, 0.0) - logp.gather(1, ids.clamp(min=0)))
        loss[rows] = temp * temp * inner.sum(1)
        if grad is not None:
            g = torch.exp(logp)
            g.scatter_add_(1, ids.clamp(min=0), -q)
            grad[rows] = g * (s["loss_grad"][rows].to(f64) * temp)[:, None]
    return (loss, lse) if grad is None else (loss, lse, grad)
