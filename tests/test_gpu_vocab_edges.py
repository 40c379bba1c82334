"""The vocabulary operators where values are not finite, near the type's limits or cancel, against their definitions in 64
bits with the bounds of test_gpu_vocab_ops."""
import threading

import numpy as np
import pytest

from gpu_util import driver, host, tuning
from test_gpu_vocab_ops import BOTH, HALF, U, Distill, Vocab, blank, near, space, values

pytestmark = pytest.mark.gpu
LOWEST = 255 * 2.0 ** 120                                      # the largest magnitude of a bf16, in both types


# ---- vocabulary loss: weights of the tokens --------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("keep", [1, 2])
@pytest.mark.parametrize("kind", ["all nan", "nan and zero", "one nan", "one inf", "inf and zero"])
def test_vocab_loss_weights_that_are_not_finite(dtype, keep, kind):
    """Such a weight reaches its own token's dx and the sums over the tokens (dw, db), and no other token's dx."""
    v = Vocab(dtype, 60, 72, 400, bias=True, ignore=-1)
    v.labels[5], v.labels[7] = 11, -1
    if "zero" in kind:
        v.gs[:] = 0.0
    v.gs[5] = np.inf if "inf" in kind else np.nan
    if kind == "all nan":
        v.gs[:] = np.nan
    v.gs[7] = np.nan                                             # an ignored token's: no part in anything
    bad = (v.labels != -1) & ~np.isfinite(v.gs)
    sound = Vocab(dtype, 60, 72, 400, bias=True, ignore=-1)
    sound.labels, sound.gs = v.labels, np.where(np.isfinite(v.gs), v.gs, 0.0).astype(np.float32)
    sound.reference()
    with tuning("vocab_keep", keep):
        for run in (v.both, lambda: (v.forward(), v.backward())):
            v.outputs()
            run()
            dx, dw, db = values(v.o_dx), values(v.o_dw), values(v.o_db)
            near(dx[~bad], sound.dx[~bad], sound.edx[~bad])
            assert not np.isfinite(dx[bad]).any() and bad[5] and not bad[7]
            assert not np.isfinite(dw).any() and not np.isfinite(db).any()


# ---- scores far from zero ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("keep", [1, 2])
def test_vocab_loss_scores_of_any_size(dtype, keep):
    """Tokens whose largest scores are 1e6 to 1e32 and whose next ones are far below: lse is the largest score, the gradient
    that of one entry against the label, and the other tokens' are as they were."""
    v = Vocab(dtype, 80, 40, 900, bias=True)
    big = {3: 1e6, 9: 3e9, 10: 3e10, 11: -7e11, 40: 2e15, 70: -1e20, 79: 1e32}
    best, worst = 500, 20                                          # the rows with the largest and the smallest first column
    v.w[:, 0] *= 0.5
    v.w[best, 0], v.w[worst, 0] = 8.0, -8.0
    for t, x in big.items():
        v.x[t] = 0.0
        v.x[t, 0] = x
        v.labels[t] = 7
    v.x64, v.w64 = values(v.x), values(v.w)
    v.gs[:] = 0.5
    v.reference()
    rows, rest = list(big), [t for t in range(80) if t not in big]
    with tuning("vocab_keep", keep):
        for run in (v.both, lambda: (v.forward(), v.backward())):
            v.outputs()
            run()
            near(values(v.o_lse)[rest], v.lse[rest], v.else_[rest])
            near(values(v.o_dx)[rest], v.dx[rest], v.edx[rest])
            # one product, the bias, a sum of one: four roundings at most
            near(values(v.o_lse)[rows], v.lse[rows], 4 * U * np.abs(v.lse[rows]))
            near(values(v.o_loss)[rows], v.loss[rows], 8 * U * np.abs(v.lse[rows]))
            # G is 1 and -1 (times the weight, which the largest of them divides: all are alike), exactly
            top = [best if x > 0 else worst for x in big.values()]
            want = 0.5 * (v.w64[top] - v.w64[7])
            near(values(v.o_dx)[rows], want, (2 * U + HALF[dtype]) * 0.5 * (np.abs(v.w64[top]) + np.abs(v.w64[7])))
            assert np.isfinite(values(v.o_dw)).all() and np.isfinite(values(v.o_db)).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("keep", [1, 2])
def test_vocab_loss_backward_from_an_lse_of_large_scores_in_another_order(dtype, keep):
    """The loss of a few tokens over odd rows adds the width up in shares; the gradient's scores may lie above its lse by their
    rounding, which is far more than 1 here.  G stays within 1."""
    v = Vocab(dtype, 16, 1211, 3000, bias=False)
    v.x *= 1e12
    v.labels[:] = np.arange(16)
    v.gs[:] = 1.0
    v.outputs()
    v.forward()
    assert driver().lib.cct_hip_last_kernel().decode().startswith("vocab_few_kernel<")
    with tuning("vocab_keep", keep):
        v.backward()
    w, x = values(v.w), values(v.x)
    dx, dw = values(v.o_dx), values(v.o_dw)
    assert np.isfinite(dx).all() and np.isfinite(dw).all()
    # |G| <= 1 in every entry; all but a handful of scores are far below the largest
    assert (np.abs(dw) <= np.abs(x).sum(0) * (1 + 2 * HALF[dtype])).all()
    assert (np.abs(dx) <= np.abs(w).sum(0) * (1 + 2 * HALF[dtype])).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("keep", [1, 2])
@pytest.mark.parametrize("tokens, width", [(70, 8), (5, 33)])
@pytest.mark.parametrize("top, rest", [(4000.0, 3984.0), (-LOWEST, -LOWEST), (-1e30, -1e30), (2.0 ** 70, 2.0 ** 70)])
def test_vocab_loss_is_not_lost_in_the_size_of_the_scores(dtype, keep, tokens, width, top, rest):
    """Scores that are the bias alone: one entry ahead of the others by 16, or all alike.  The loss is of the size of the
    scores' differences, whatever their own."""
    v = Vocab(dtype, tokens, width, 900, bias=True)
    v.x[:] = 0.0
    v.b[:] = rest
    v.b[123] = top
    v.labels[:] = np.where(np.arange(tokens) % 3 == 0, 123, 7)
    b = values(v.b)
    ahead = float(b[123] - b[7])
    assert ahead in (0.0, 16.0)
    log_sum = np.log1p(899 * np.exp(-ahead))
    want = np.where(v.labels == 123, log_sum, log_sum + ahead)
    with tuning("vocab_keep", keep):
        for run in (v.forward, v.both):
            v.outputs()
            run()
            # exponentials and their sum: at most 100 additions in a row onto it; the logarithm and the difference in the result
            near(values(v.o_loss), want, 100 * U + 2.0 ** -21 + 2 * U * want)
            near(values(v.o_lse), np.full(tokens, b[123] + log_sum), 4 * U * abs(top))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("vocab", [300, 9001, 140000])
@pytest.mark.parametrize("temperature", [1.0, 2.0, 0.25])
@pytest.mark.parametrize("level", [-LOWEST, 4000.0, -1e30])
def test_distill_loss_is_not_lost_in_the_size_of_the_scores(dtype, vocab, temperature, level):
    """Scores that are all alike, at any level: the student's distribution is uniform."""
    d = Distill(dtype, 3, vocab, 4, temperature=temperature)
    d.z[:] = level
    d.ids[:] = [0, 5, vocab - 1, -1]
    d.tl[:] = np.array([1.0, 2.0, 0.0, 9.0]) * temperature
    d.upload()
    q = np.exp([1.0, 2.0, 0.0])
    q /= q.sum()
    want = temperature ** 2 * (q * (np.log(q) + np.log(vocab))).sum()
    for both in (False, True):
        d.run(both)
        # additions as in Distill.reference, and the roundings of a sum of terms of log(vocab)
        bound = temperature ** 2 * ((vocab / 256 + 200) * U * 2 + 20 * U * np.log(vocab) + 2.0 ** -20)
        near(values(d.o_loss), np.full(3, want), bound)


@pytest.mark.parametrize("dtype, tokens, vocab", [(d, 3, v) for d in BOTH for v in (300, 9001, 140000)] + [("bf16", 8200, 140000)])
@pytest.mark.parametrize("temperature, level", [(1.5, 1e10), (1.5, -LOWEST), (0.3, -1e30), (3.0, 4000.0)])
def test_distill_gradient_of_scores_of_any_size(dtype, tokens, vocab, temperature, level):
    """Scores that are all alike, at any level: p is 1 / vocab.  From the lse alone it is known to 2^-23 |lse|, and at most 1."""
    import torch
    d = Distill(dtype, 3, vocab, 4, temperature=temperature)
    if tokens > 3:                                                 # more tokens than rows are cut into ranges for
        d.z = torch.empty((tokens, vocab), dtype=torch.bfloat16, device="cuda")
    d.z[:] = level
    d.tokens = tokens
    d.ids = np.tile([0, 5, vocab - 1, -1], (tokens, 1))
    d.tl = np.tile(np.array([1.0, 2.0, 0.0, 9.0]) * temperature, (tokens, 1)).astype(np.float32)
    d.gs = np.full(tokens, 0.5, np.float32)
    d.upload()
    q = np.exp([1.0, 2.0, 0.0])
    want = np.full(vocab, 1.0 / vocab)
    want[[0, 5, vocab - 1]] -= q / q.sum()
    want *= 0.5 * temperature
    d.run(True)
    # p: the sum's additions (as in Distill.reference), its logarithm, the exponential; q: four entries; the products
    e = ((vocab / 256 + 200) * U * 2 + 8 * U * np.log(vocab) + 2.0 ** -20) / vocab
    bound = 0.5 * temperature * (e + (want < 0) * (16 * U + 2.0 ** -20)) + 4 * U * np.abs(want)
    bound += HALF[dtype] * (np.abs(want) + bound)
    some = d.o_d if tokens == 3 else d.o_d[[0, 1, tokens // 2, tokens - 1]]
    near(values(some), np.tile(want, (some.shape[0], 1)), np.tile(bound, (some.shape[0], 1)))
    d.run(False)
    some = values(d.o_d if tokens == 3 else d.o_d[[0, 1, tokens // 2, tokens - 1]])
    most = 0.5 * temperature * (1 + 2.0 ** -20) * (1 + HALF[dtype])
    assert (np.abs(some) <= most).all()
    lse = abs(level) / temperature + np.log(vocab)
    if lse * 2.0 ** -23 < 0.01:
        worse = 0.5 * temperature / vocab * 2.1 * lse * 2.0 ** -23
        near(some, np.tile(want, (some.shape[0], 1)), np.tile(bound + worse * (1 + HALF[dtype]), (some.shape[0], 1)))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("vocab", [300, 9001])
@pytest.mark.parametrize("temperature", [2.0 ** -60, 2.0 ** 60])
def test_distill_loss_at_the_ends_of_the_temperatures(dtype, vocab, temperature):
    """Cold: all of p on the largest score and of q on the teacher's largest.  Hot: both uniform."""
    d = Distill(dtype, 2, vocab, 3, temperature=temperature)
    d.z[:] = 0.0
    d.z[:, 8] = 1.0
    d.ids = np.tile([8, 20, -1], (2, 1))
    d.tl = np.tile([0.5, 0.25, 9.0], (2, 1)).astype(np.float32)
    d.gs = np.full(2, 1.0, np.float32)
    d.upload()
    cold = temperature < 1
    want = np.zeros(vocab) if cold else np.full(vocab, 1.0 / vocab)
    if not cold:
        want[[8, 20]] -= 0.5
    for both in (False, True):
        d.run(both)
        loss = 0.0 if cold else temperature ** 2 * np.log(vocab / 2)
        near(values(d.o_loss), np.full(2, loss), abs(loss) * ((vocab / 256 + 200) * U * 2 + 2.0 ** -20))
        near(values(d.o_d) / temperature, np.tile(want, (2, 1)),
             ((vocab / 256 + 200) * U * 2 + 40 * U * np.log(vocab) + 2.0 ** -20 + 1.1 * HALF[dtype]) * np.tile(np.abs(want), (2, 1)))


# ---- knobs that change while calls run ---------------------------------------------------------------------------------
@pytest.mark.parametrize("training", [False, True])
def test_vocab_loss_while_another_thread_changes_its_tile(training):
    """A call keeps to the tile that it began with: every result is that of one setting or of the other, and the workspace,
    which has room for either, ends where it says."""
    import torch
    from caffecontroll_amd.driver import BF16, vocab_loss_args
    drv, tokens, width, vocab = driver(), 1023, 64, 50021
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, w = (torch.randn(n, width, generator=gen, device="cuda").to(torch.bfloat16) for n in (tokens, vocab))
    labels = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    a, need = vocab_loss_args(tokens, width, vocab, BF16), 0
    for tile in (0, 3):
        with tuning("vocab_tile", tile):
            need = max(need, drv.vocab_loss_workspace_bytes(a, training))
    ws = space(need)

    def outputs():
        o = [blank((tokens,)), blank((tokens,))]
        return o + [blank(x.shape, "bf16"), blank(w.shape, "bf16")] if training else o

    def call(o):
        if training:
            drv.vocab_loss_forward_backward(o[0], o[1], o[2], o[3], None, x, w, None, labels, None, a, ws.ptr, need)
        else:
            drv.vocab_loss_forward(o[0], o[1], x, w, None, labels, a, ws.ptr, need)

    want = []
    for tile in (0, 3):
        with tuning("vocab_tile", tile):
            o = outputs()
            call(o)
            want.append([host(t.float()) for t in o])
    stop = threading.Event()

    def change():
        n = 0
        while not stop.is_set():
            n += 1
            drv.set_tuning("vocab_tile", 3 * (n % 2))

    other = threading.Thread(target=change)
    other.start()
    try:
        got = []
        for _ in range(60):
            o = outputs()
            call(o)
            got.append([host(t.float()) for t in o])
    finally:
        stop.set()
        other.join()
        drv.set_tuning("vocab_tile", 0)
    assert ws.intact()
    for g in got:
        assert any(all(np.array_equal(a, b) for a, b in zip(g, w)) for w in want)
