"""The vocabulary operators as a model uses them: a token model whose embedding is also its output matrix, trained and
distilled with the driver's inner-product and update entry points around them; the same calls in captured graphs, on other
streams, and with arrays whose offsets pass 32 bits."""
import numpy as np
import pytest

from gpu_util import driver, host, rel_err

pytestmark = pytest.mark.gpu
N_, T_ = 111, 112


def cuda(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a))
    return t.to(dtype).cuda() if dtype else t.cuda()


def workspace(n):
    import torch
    return torch.full((max(16, n),), 0xFF, dtype=torch.uint8, device="cuda")


class Model:
    """ids -> scale * E[ids] -> ReLU(inner product) -> scores with E again, fp32, on the driver's entry points."""

    def __init__(self, tokens=60, width=48, vocab=310, seed=0):
        import torch
        from caffecontroll_amd.driver import distill_loss_args, embedding_args, vocab_loss_args
        rng = np.random.default_rng(seed)
        self.n, self.h, self.v, self.drv = tokens, width, vocab, driver()
        self.scale = 3.0
        self.E = (rng.standard_normal((vocab, width)) / np.sqrt(width)).astype(np.float32)
        self.W = (rng.standard_normal((width, width)) / np.sqrt(width)).astype(np.float32)
        self.b, self.ob = (rng.standard_normal(k).astype(np.float32) * 0.1 for k in (width, vocab))
        self.ids = np.minimum(rng.zipf(1.4, tokens) - 1, vocab - 1).astype(np.int32)
        self.labels = rng.integers(0, vocab, tokens).astype(np.int32)
        self.ids[3], self.labels[[5, 6]] = -1, -1
        self.gs = np.full(tokens, 1.0 / tokens, np.float32)
        self.d = {k: cuda(getattr(self, k)) for k in ("E", "W", "b", "ob", "ids", "labels", "gs")}
        for name, shape in dict(e=(tokens, width), hid=(tokens, width), dhid=(tokens, width), dpre=(tokens, width),
                                de=(tokens, width), dE=(vocab, width), dob=(vocab,), dW=(width, width), db=(width,),
                                loss=(tokens,), lse=(tokens,), scores=(tokens, vocab), dscores=(tokens, vocab),
                                hE=(vocab, width), hW=(width, width)).items():
            self.d[name] = torch.full(shape, float("nan"), device="cuda")
        self.d["hE"].zero_()
        self.d["hW"].zero_()
        k = 7
        self.top_ids = np.stack([rng.permutation(vocab)[:k] for _ in range(tokens)]).astype(np.int32)
        self.top = rng.standard_normal((tokens, k)).astype(np.float32)
        self.d["top_ids"], self.d["top"] = cuda(self.top_ids), cuda(self.top)
        self.ea = embedding_args(tokens, width, vocab, scale=self.scale)
        self.va = vocab_loss_args(tokens, width, vocab)
        self.da = distill_loss_args(tokens, vocab, k, temperature=1.5)
        self.bytes = max(self.drv.embedding_workspace_bytes(self.ea), self.drv.vocab_loss_workspace_bytes(self.va),
                         self.drv.distill_loss_workspace_bytes(self.da))
        self.space = workspace(self.bytes)

    def hidden(self):
        d, n, h = self.d, self.n, self.h
        self.drv.embedding_forward(d["e"], d["E"], d["ids"], self.ea)
        self.drv.sgemm_new_bias(N_, T_, n, h, h, 1.0, d["e"], d["W"], 0.0, d["hid"], d["b"], relu=True)

    def below(self):
        """From dhid to the gradients of the inner product and, on top of the output matrix's, of the embedding."""
        d, n, h = self.d, self.n, self.h
        self.drv.relu_backward(d["dpre"], d["dhid"], d["hid"], n * h)
        self.drv.sgemm_new_colsum(T_, N_, h, h, n, 1.0, d["dpre"], d["e"], 0.0, d["dW"], d["db"], d["dpre"], n, h)
        self.drv.sgemm_new(N_, N_, n, h, h, 1.0, d["dpre"], d["W"], 0.0, d["de"])
        self.drv.embedding_backward(d["dE"], d["de"], d["ids"], self.ea, self.space, self.bytes, accumulate=True)

    def train_step(self):
        d = self.d
        self.hidden()
        self.drv.vocab_loss_forward_backward(d["loss"], d["lse"], d["dhid"], d["dE"], d["dob"], d["hid"], d["E"], d["ob"],
                                             d["labels"], d["gs"], self.va, self.space, self.bytes)
        self.below()

    def distill_step(self):
        d, n, h, v = self.d, self.n, self.h, self.v
        self.hidden()
        self.drv.sgemm_new_bias(N_, T_, n, v, h, 1.0, d["hid"], d["E"], 0.0, d["scores"], d["ob"])
        self.drv.distill_loss_forward_backward(d["loss"], d["lse"], d["dscores"], d["scores"], d["top_ids"], d["top"],
                                               d["gs"], self.da, self.space, self.bytes)
        self.drv.sgemm_new(N_, N_, n, h, v, 1.0, d["dscores"], d["E"], 0.0, d["dhid"])
        self.drv.sgemm_new(T_, N_, v, h, n, 1.0, d["dscores"], d["hid"], 0.0, d["dE"])
        self.below()

    def reference(self, distill):
        import torch
        p = {k: torch.from_numpy(getattr(self, k)).double().requires_grad_() for k in ("E", "W", "b", "ob")}
        ids, labels = torch.from_numpy(self.ids).long(), torch.from_numpy(self.labels).long()
        e = torch.where((ids >= 0)[:, None], self.scale * p["E"][ids.clamp(min=0)], torch.zeros((), dtype=torch.float64))
        scores = torch.relu(e @ p["W"].T + p["b"]) @ p["E"].T + p["ob"]
        gs = torch.from_numpy(self.gs).double()
        if distill:
            t = 1.5
            logq = torch.log_softmax(torch.from_numpy(self.top).double() / t, 1)
            logp = torch.log_softmax(scores / t, 1).gather(1, torch.from_numpy(self.top_ids).long())
            loss = t * t * (logq.exp() * (logq - logp)).sum(1)
        else:
            logp = torch.log_softmax(scores, 1).gather(1, labels.clamp(min=0)[:, None])[:, 0]
            loss = torch.where(labels >= 0, -logp, torch.zeros((), dtype=torch.float64))
        (loss * gs).sum().backward()
        return loss.detach().numpy(), {k: t.grad.numpy() for k, t in p.items() if t.grad is not None}


# at most 310 terms a sum, four products behind one another: 4 * 310 * 2^-24 = 7e-5 of the largest value
BAR = 1e-4


@pytest.mark.parametrize("distill", [False, True])
@pytest.mark.parametrize("tokens, width, vocab", [(1, 8, 300), (60, 48, 310), (130, 36, 257)])
def test_tied_model_gradients(distill, tokens, width, vocab):
    m = Model(max(tokens, 8), width, vocab)
    m.distill_step() if distill else m.train_step()
    loss, g = m.reference(distill)
    assert rel_err(host(m.d["loss"]), loss) <= BAR
    names = dict(E="dE", W="dW", b="db") if distill else dict(E="dE", W="dW", b="db", ob="dob")
    for k, name in names.items():
        assert rel_err(host(m.d[name]), g[k]) <= BAR, name


def test_training_steps_update_the_tied_matrix():
    """Three steps with the driver's update: every step's gradients are those of the weights it saw."""
    m = Model(40, 32, 300, seed=4)
    for _ in range(3):
        m.E, m.W = host(m.d["E"]).copy(), host(m.d["W"]).copy()
        m.train_step()
        _, g = m.reference(False)
        assert rel_err(host(m.d["dE"]), g["E"]) <= BAR and rel_err(host(m.d["dW"]), g["W"]) <= BAR
        m.drv.sgd_update_batch([(m.d["E"].numel(), m.d["E"], m.d["dE"], m.d["hE"], 0.1, 0.9, 0.0, False),
                                (m.d["W"].numel(), m.d["W"], m.d["dW"], m.d["hW"], 0.1, 0.9, 0.0, False)])
        assert not np.array_equal(host(m.d["E"]), m.E)


# ---- graphs and streams ------------------------------------------------------------------------------------------------
def capture(fn):
    """fn() once eagerly on a side stream, then under capture there."""
    import torch
    drv, main, side, graph = driver(), torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(main)
    try:
        with torch.cuda.stream(side):
            drv.set_stream(side.cuda_stream)
            fn()
            side.synchronize()
            with torch.cuda.graph(graph, stream=side):
                fn()
    finally:
        drv.set_stream(main.cuda_stream)
    torch.cuda.synchronize()
    return graph


def poison(tensors):
    for t in tensors:
        t.fill_(float("nan"))


def bf16_calls(seed, tokens, width, vocab, top):
    """One call of every entry point in bf16 with outputs and a workspace of its own: (function, outputs)."""
    import torch
    from caffecontroll_amd.driver import BF16, distill_loss_args, embedding_args, vocab_loss_args
    drv, g = driver(), torch.Generator(device="cuda")
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    x, w, bias = rnd(tokens, width), rnd(vocab, width) * width ** -0.5, rnd(vocab)
    ids = torch.randint(0, vocab // 8, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    labels = torch.randint(0, vocab, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    top_ids = torch.randint(0, vocab, (tokens, top), generator=g, device="cuda", dtype=torch.int32)
    weights, scores = torch.randn(tokens, top, generator=g, device="cuda"), rnd(tokens, vocab)
    gs = torch.rand(tokens, generator=g, device="cuda")
    ea, va = embedding_args(tokens, width, vocab, BF16, 0.5), vocab_loss_args(tokens, width, vocab, BF16)
    da = distill_loss_args(tokens, vocab, top, BF16, 2.0)
    n = max(drv.embedding_workspace_bytes(ea), drv.vocab_loss_workspace_bytes(va), drv.distill_loss_workspace_bytes(da))
    space = workspace(n)
    o = dict(e=torch.empty_like(x), de=torch.empty_like(w), loss=torch.empty(tokens, device="cuda"),
             lse=torch.empty(tokens, device="cuda"), dx=torch.empty_like(x), dw=torch.empty_like(w), db=torch.empty_like(bias),
             dx2=torch.empty_like(x), dw2=torch.empty_like(w), dl=torch.empty(tokens, device="cuda"),
             dlse=torch.empty(tokens, device="cuda"), ds=torch.empty_like(scores), ds2=torch.empty_like(scores))

    def run():
        drv.embedding_forward(o["e"], w, ids, ea)
        drv.embedding_backward(o["de"], x, ids, ea, space, n)
        drv.vocab_loss_forward_backward(o["loss"], o["lse"], o["dx"], o["dw"], o["db"], x, w, bias, labels, gs, va, space, n)
        drv.vocab_loss_forward(o["loss"], o["lse"], x, w, bias, labels, va, space, n)
        drv.vocab_loss_backward(o["dx2"], o["dw2"], None, x, w, bias, labels, o["lse"], gs, va, space, n)
        drv.distill_loss_forward_backward(o["dl"], o["dlse"], o["ds"], scores, top_ids, weights, gs, da, space, n)
        drv.distill_loss_backward(o["ds2"], scores, top_ids, weights, o["dlse"], gs, da, space, n)
    keep = (x, w, bias, ids, labels, top_ids, weights, scores, gs, space)
    return run, list(o.values()), keep


def bits(tensors):
    return [host(t.float()).copy() for t in tensors]


@pytest.mark.parametrize("tokens, width, vocab, top", [(20, 64, 900, 5), (300, 136, 3000, 40), (9000, 16, 520, 3)])
def test_every_call_in_a_replayed_graph(tokens, width, vocab, top):
    import torch
    run, outs, _keep = bf16_calls(1, tokens, width, vocab, top)
    run()
    want = bits(outs)
    assert all(np.isfinite(w).all() for w in want)
    graph = capture(run)
    for _ in range(3):
        poison(outs)
        torch.randn(1 << 20, device="cuda").sum().item()           # eager work of the program's own
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(bits(outs), want):
            np.testing.assert_array_equal(got, w)


@pytest.mark.parametrize("tokens, width, vocab, top", [(12, 99, 40001, 5), (1023, 520, 17011, 4)])
def test_every_call_in_a_replayed_graph_few_tokens_and_rows_past_whole_rounds(tokens, width, vocab, top):
    test_every_call_in_a_replayed_graph(tokens, width, vocab, top)


def test_two_graphs_and_eager_calls_between_them():
    import torch
    a, outs_a, _ka = bf16_calls(2, 130, 72, 1100, 9)
    b, outs_b, _kb = bf16_calls(3, 40, 256, 2600, 17)
    c, outs_c, _kc = bf16_calls(4, 700, 40, 5000, 2)
    a(), b(), c()
    want = [bits(o) for o in (outs_a, outs_b, outs_c)]
    ga, gb = capture(a), capture(b)
    for order in ((ga, gb), (gb, ga), (ga, gb)):
        for o in (outs_a, outs_b, outs_c):
            poison(o)
        order[0].replay()
        c()
        order[1].replay()
        torch.cuda.synchronize()
        for o, w in zip((outs_a, outs_b, outs_c), want):
            for got, x in zip(bits(o), w):
                np.testing.assert_array_equal(got, x)


def test_calls_on_another_stream_than_the_one_before():
    import torch
    drv, main, side = driver(), torch.cuda.current_stream(), torch.cuda.Stream()
    run, outs, _keep = bf16_calls(5, 77, 88, 1500, 6)
    run()
    want = bits(outs)
    poison(outs)
    side.wait_stream(main)
    try:
        drv.set_stream(side.cuda_stream)
        run()
        side.synchronize()
    finally:
        drv.set_stream(main.cuda_stream)
    for got, w in zip(bits(outs), want):
        np.testing.assert_array_equal(got, w)


# ---- offsets past 32 bits ------------------------------------------------------------------------------------------------
def test_embedding_table_past_four_gib():
    import torch
    from caffecontroll_amd.driver import BF16, embedding_args
    drv, vocab, width, tokens = driver(), 1 << 20, 2304, 300                # 4.8 GB, 2.4e9 elements
    table = torch.zeros((vocab, width), dtype=torch.bfloat16, device="cuda")
    ids = torch.arange(vocab - tokens, vocab, device="cuda", dtype=torch.int32)
    rows = torch.randn(tokens, width, device="cuda").to(torch.bfloat16)
    table[vocab - tokens:] = rows
    out = torch.empty((tokens, width), dtype=torch.bfloat16, device="cuda")
    a = embedding_args(tokens, width, vocab, BF16)
    drv.embedding_forward(out, table, ids, a)
    assert torch.equal(out, rows)
    n = drv.embedding_workspace_bytes(a)
    table.fill_(1.0)
    drv.embedding_backward(table, rows, ids, a, workspace(n), n)
    assert torch.equal(table[vocab - tokens:], rows)
    assert not table[:vocab - tokens].any()


def test_vocab_loss_weights_past_four_gib():
    """The last rows of a matrix of 2.3e9 elements: scores, and both gradients, through several pieces."""
    import torch
    from caffecontroll_amd.driver import BF16, vocab_loss_args
    drv, vocab, width, tokens = driver(), 565000, 4096, 24
    w = torch.zeros((vocab, width), dtype=torch.bfloat16, device="cuda")
    x = torch.randn(tokens, width, device="cuda").to(torch.bfloat16)
    tail = (torch.randn(64, width, device="cuda") / 16).to(torch.bfloat16)
    w[vocab - 64:] = tail
    labels = torch.arange(vocab - tokens, vocab, device="cuda", dtype=torch.int32)
    a = vocab_loss_args(tokens, width, vocab, BF16)
    n = drv.vocab_loss_workspace_bytes(a)
    loss, lse = torch.empty(tokens, device="cuda"), torch.empty(tokens, device="cuda")
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    drv.vocab_loss_forward_backward(loss, lse, dx, dw, None, x, w, None, labels, None, a, workspace(n), n)
    s = x.double() @ tail.double().T
    total = torch.exp(s).sum(1) + (vocab - 64)
    want_lse = torch.log(total)
    at = s.gather(1, (labels.long() - (vocab - 64))[:, None])[:, 0]
    # scores of a few hundred: 4096 terms of a fp32 sum, 4096 * 2^-24 = 2.4e-4 of the terms' size
    assert float((lse.double() - want_lse).abs().max()) <= 2.4e-4 * float((x.double().abs() @ tail.double().abs().T).max())
    assert rel_err(host(loss), host(want_lse - at)) <= 2.4e-4
    g = torch.exp(s - want_lse[:, None])
    g[torch.arange(tokens), labels.long() - (vocab - 64)] -= 1.0
    # G and the result rounded to bf16, half a step each
    assert rel_err(host(dx.double()), host(g @ tail.double())) <= 2 * 2.0 ** -8
    assert rel_err(host(dw[vocab - 64:].double()), host(g.T @ x.double())) <= 2 * 2.0 ** -8
    rest = (1.0 / total)[:, None] * x.double()
    assert rel_err(host(dw[5].double()), host(rest.sum(0))) <= 2 * 2.0 ** -8


@pytest.mark.parametrize("tokens, width", [(8, 4095), (80, 4096)])
def test_vocab_loss_alone_past_four_gib(tokens, width):
    """The loss of few tokens over rows of an odd length, and the loss of more as one piece of 565000 rows."""
    import torch
    from caffecontroll_amd.driver import BF16, vocab_loss_args
    drv, vocab = driver(), 565000
    w = torch.zeros((vocab, width), dtype=torch.bfloat16, device="cuda")
    x = torch.randn(tokens, width, device="cuda").to(torch.bfloat16)
    tail = (torch.randn(64, width, device="cuda") / 16).to(torch.bfloat16)
    w[vocab - 64:] = tail
    labels = torch.arange(vocab - tokens, vocab, device="cuda", dtype=torch.int32).clamp_(min=vocab - 64)
    a = vocab_loss_args(tokens, width, vocab, BF16)
    n = drv.vocab_loss_workspace_bytes(a, training=False)
    loss, lse = torch.empty(tokens, device="cuda"), torch.empty(tokens, device="cuda")
    drv.vocab_loss_forward(loss, lse, x, w, None, labels, a, workspace(n), n)
    s = x.double() @ tail.double().T
    want_lse = torch.log(torch.exp(s).sum(1) + (vocab - 64))
    at = s.gather(1, (labels.long() - (vocab - 64))[:, None])[:, 0]
    # width terms of a fp32 sum, as above; lse and the label's score each
    size = 2.5e-4 * float((x.double().abs() @ tail.double().abs().T).max())
    assert float((lse.double() - want_lse).abs().max()) <= size
    assert float((loss.double() - (want_lse - at)).abs().max()) <= 2 * size


def test_distill_scores_past_four_gib():
    import torch
    from caffecontroll_amd.driver import BF16, distill_loss_args
    drv, tokens, vocab = driver(), 18000, 131072                             # 4.7 GB
    z = torch.zeros((tokens, vocab), dtype=torch.bfloat16, device="cuda")
    last = torch.randn(vocab, device="cuda").to(torch.bfloat16)
    z[-1] = last
    ids = torch.zeros((tokens, 2), dtype=torch.int32, device="cuda")
    ids[:, 1] = vocab - 1
    top = torch.zeros((tokens, 2), device="cuda")
    a = distill_loss_args(tokens, vocab, 2, BF16)
    n = drv.distill_loss_workspace_bytes(a)
    loss, lse = torch.empty(tokens, device="cuda"), torch.empty(tokens, device="cuda")
    drv.distill_loss_forward_backward(loss, lse, z, z, ids, top, None, a, workspace(n), n)   # in place
    want = torch.softmax(last.double(), 0)
    want[0] -= 0.5
    want[-1] -= 0.5
    assert rel_err(host(z[-1].double()), host(want)) <= 1.01 * 2.0 ** -8
    assert rel_err(host(z[-2, 1:9].double()), np.full(8, 1.0 / vocab)) <= 1.01 * 2.0 ** -8
    assert abs(float(lse[-1]) - float(torch.logsumexp(last.double(), 0))) <= 1e-5 * 13
    assert abs(float(loss[0]) - np.log(vocab / 2)) <= 1e-5 * 13
