"""Embedding, vocabulary loss and distillation loss against their definitions in 64 bits.

Tolerances are worst-case bounds of the arithmetic, computed beside each reference: u = 2^-24 is half a step of fp32, and a
result stored as T is off by at most half a step of T on top.  n additions of terms t in fp32 are off by at most
n * u * sum |t|; an exponential by ln 2 * (error of its exponent) + 2^-22 (a rounding of the argument's product with
log2 e, and the instruction's own step)."""
import numpy as np
import pytest

from gpu_util import driver, host, tuning

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TINY = 2.0 ** -126
HALF = {"f32": U, "bf16": 2.0 ** -8}
BOTH = ("f32", "bf16")


def torch_type(dtype):
    import torch
    return torch.bfloat16 if dtype == "bf16" else torch.float32


def code(dtype):
    from caffecontroll_amd.driver import BF16, F32
    return BF16 if dtype == "bf16" else F32


def up(a, dtype="f32", stride=0, fill=float("nan")):
    """The array on the device in its type, its rows `stride` elements apart with `fill` between them; and the values that
    it holds, in 64 bits."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(torch_type(dtype))
    if stride:
        whole = torch.full((a.shape[0], stride), fill, dtype=t.dtype)
        whole[:, :a.shape[1]] = t
        return whole.cuda(), t.double().numpy()
    return t.cuda(), t.double().numpy()


def ints(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def blank(shape, dtype="f32", fill=float("nan")):
    import torch
    return torch.full(shape, fill, dtype=torch_type(dtype), device="cuda")


def space(n):
    """A workspace that holds garbage (NaN in every type) and ends where it says: the 4 KB behind it stay as they are."""
    import torch
    n = (n + 15) // 16 * 16
    whole = torch.full((n + 4096,), 0xFF, dtype=torch.uint8, device="cuda")

    class Space:
        ptr = whole.data_ptr()

        @staticmethod
        def intact():
            return bool((whole[n:] == 0xFF).all())
    return Space


def values(t):
    return host(t.double())


def near(got, want, bound):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= bound) & ~(np.isnan(got) & np.isnan(want)) & ~(got == want)
    assert not bad.any(), "%d of %d off, first at %s: %r, expected %r within %r" % (
        bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], want[bad][0], np.broadcast_to(bound, got.shape)[bad][0])


# ---- embedding ---------------------------------------------------------------------------------------------------
def embedding_rows(ids, vocab, pad):
    return (ids != pad) & (ids >= 0) & (ids < vocab)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("tokens, width, vocab, gap", [
    (1, 1, 1, 0), (1, 4096, 50, 0), (3, 7, 11, 0), (8, 64, 100, 0), (65, 130, 33, 5), (300, 1001, 500, 0),
    (517, 2048, 1000, 8), (2500, 33, 7, 1)])
def test_embedding_forward(dtype, tokens, width, vocab, gap):
    from caffecontroll_amd.driver import embedding_args
    drv, rng = driver(), np.random.default_rng(tokens + width)
    stride = width + gap if gap else 0
    table, t64 = up(rng.standard_normal((vocab, width)), dtype, stride)
    ids = rng.integers(0, vocab, tokens)
    ids[rng.random(tokens) < 0.1] = -1
    ids[0] = vocab - 1
    if tokens > 60:
        ids[7], ids[8], ids[9] = vocab, -2, 2 ** 31 - 1        # named rows that do not exist
    out = blank((tokens, stride or width), dtype, 3.0)
    scale = 1.7
    drv.embedding_forward(out, table, ids_dev := ints(ids), embedding_args(tokens, width, vocab, code(dtype), scale, -1,
                                                                           stride, stride))
    got, ok = values(out), embedding_rows(ids, vocab, -1)
    s32 = float(np.float32(scale))
    want = np.where(ok[:, None], s32 * t64[np.where(ok, ids, 0)], np.where(ids == -1, 0.0, np.nan)[:, None])
    # a product in fp32 and a rounding to the type
    near(got[:, :width], want, np.abs(want) * (U + HALF[dtype] * (1 + U)))
    assert (got[:, width:] == 3.0).all()
    assert (host(ids_dev) == ids).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("tokens, width, vocab, kind", [
    (1, 5, 3, "uniform"), (64, 8, 4, "one"), (128, 1030, 40, "skewed"), (127, 6, 1000, "uniform"), (128, 2060, 7, "one"), (65, 8, 4, "one"), (129, 33, 9, "one"), (200, 64, 1000, "uniform"),
    (640, 12, 3, "uniform"), (1000, 130, 50, "skewed"), (4099, 40, 10007, "skewed"), (8192, 4, 513, "uniform"),
    (8193, 20, 600, "skewed"), (20000, 9, 300000, "uniform"), (30000, 16, 511, "skewed"), (12345, 8, 512, "one"),
    (9000, 3, 40, "padding")])
def test_embedding_backward(dtype, accumulate, tokens, width, vocab, kind):
    from caffecontroll_amd.driver import embedding_args
    drv, rng = driver(), np.random.default_rng(tokens * 7 + width)
    gap = 3 if width in (33, 130, 20) else 0
    stride = width + gap if gap else 0
    if kind == "one":
        ids = np.full(tokens, vocab // 2)
    elif kind == "skewed":
        ids = np.minimum(rng.zipf(1.3, tokens) - 1, vocab - 1)
    else:
        ids = rng.integers(0, vocab, tokens)
    pad = -1
    if kind == "padding":
        pad = 17                                               # a row of the table that takes no gradient
        ids[rng.random(tokens) < 0.5] = pad
    elif tokens > 100 and kind != "one":
        ids[5], ids[50], ids[60], ids[61] = -1, vocab, -7, vocab + 5
    dout, d64 = up(rng.standard_normal((tokens, width)), dtype, stride)
    old, o64 = up(rng.standard_normal((vocab, width)), dtype, stride, 3.0)
    args = embedding_args(tokens, width, vocab, code(dtype), 0.3, pad, stride, stride)
    n = drv.embedding_workspace_bytes(args)
    ws = space(n)
    drv.embedding_backward(old, dout, ints(ids), args, ws.ptr, n, accumulate)
    got = values(old)
    assert ws.intact()
    s32 = float(np.float32(0.3))
    ok = embedding_rows(ids, vocab, pad)
    total, size, count = np.zeros((vocab, width)), np.zeros((vocab, width)), np.zeros(vocab)
    np.add.at(total, ids[ok], d64[ok])
    np.add.at(size, ids[ok], np.abs(d64[ok]))
    np.add.at(count, ids[ok], 1)
    want = s32 * total + (o64 if accumulate else 0.0)
    # count additions, the product with the scale, the addition to what was there, the rounding to the type
    bound = s32 * (count[:, None] + 1) * U * size * (1 + 1e-3) + (U * np.abs(want) if accumulate else 0)
    near(got[:, :width], want, bound + HALF[dtype] * (np.abs(want) + bound))
    if gap:
        assert (got[:, width:] == 3.0).all()
    if accumulate:
        assert (got[:, :width][count == 0] == o64[count == 0]).all()


@pytest.mark.parametrize("tokens", [100, 200, 9000])
def test_embedding_backward_clears_more_rows_with_gaps_than_a_launch_has_workgroups(tokens):
    import torch
    from caffecontroll_amd.driver import embedding_args
    drv, rng, vocab = driver(), np.random.default_rng(tokens), (1 << 24) + 77
    ids = rng.permutation(vocab - 1)[:tokens]
    ids[0] = vocab - 1
    dout, d64 = up(rng.standard_normal((tokens, 1)))
    table = blank((vocab, 2), fill=3.0)
    args = embedding_args(tokens, 1, vocab, table_stride=2)
    n = drv.embedding_workspace_bytes(args)
    drv.embedding_backward(table, dout, ints(ids), args, space(n).ptr, n)
    assert bool((table[:, 1] == 3.0).all())
    at = torch.from_numpy(ids).cuda()
    np.testing.assert_array_equal(values(table[at, 0]), d64[:, 0])     # one token a row, a scale of 1: exact
    table[at, 0] = 0.0
    assert int(torch.count_nonzero(table[:, 0])) == 0


def test_embedding_backward_is_the_same_every_time_and_clears_without_tokens():
    import torch
    from caffecontroll_amd.driver import embedding_args
    drv, rng = driver(), np.random.default_rng(3)
    ids = ints(np.minimum(rng.zipf(1.2, 20000) - 1, 999))
    dout, _ = up(rng.standard_normal((20000, 32)))
    args = embedding_args(20000, 32, 1000)
    n = drv.embedding_workspace_bytes(args)
    first = None
    for _ in range(3):
        out = blank((1000, 32))
        drv.embedding_backward(out, dout, ids, args, space(n).ptr, n)
        first = host(out) if first is None else first
        np.testing.assert_array_equal(host(out), first)
    empty = embedding_args(0, 32, 1000)
    out = blank((1000, 32))
    drv.embedding_backward(out, None, None, empty, None, 0)
    assert (host(out) == 0).all()
    out.fill_(2.0)
    drv.embedding_backward(out, None, None, empty, None, 0, accumulate=True)
    drv.embedding_forward(None, None, None, empty)
    assert (host(out) == 2.0).all()
    assert torch.cuda.current_device() == 0


# ---- vocabulary loss -----------------------------------------------------------------------------------------------
class Vocab:
    """One problem, its result in 64 bits and the bounds of the arithmetic."""

    def __init__(self, dtype, tokens, width, vocab, bias, seed=0, ignore=-1, gap=0, peaked=False):
        rng = np.random.default_rng(seed + tokens * 3 + width * 5 + vocab)
        self.dtype, self.tokens, self.width, self.vocab, self.ignore = dtype, tokens, width, vocab, ignore
        self.xs, self.ws = (width + gap if gap else 0), (width + 2 * gap if gap else 0)
        w = rng.standard_normal((vocab, width)) / np.sqrt(width)
        labels = rng.integers(0, vocab, tokens)
        x = rng.standard_normal((tokens, width)) * 2 + (np.sqrt(width) * 3 * w[labels] if peaked else 0)
        if tokens > 3:
            labels[rng.random(tokens) < 0.15] = ignore
            labels[tokens // 2] = vocab - 1
        self.labels = labels
        self.x, self.x64 = up(x, dtype, self.xs)
        self.w, self.w64 = up(w, dtype, self.ws)
        self.b, self.b64 = up(rng.standard_normal(vocab), dtype) if bias else (None, np.zeros(vocab))
        self.gs = rng.random(tokens).astype(np.float32) + 0.1
        self.gs[rng.random(tokens) < 0.1] = 0.0

    def args(self, piece=0):
        from caffecontroll_amd.driver import vocab_loss_args
        return vocab_loss_args(self.tokens, self.width, self.vocab, code(self.dtype), self.ignore, piece, self.xs, self.ws)

    def reference(self):
        live = self.labels != self.ignore
        named = live & (self.labels >= 0) & (self.labels < self.vocab)
        at = np.where(named, self.labels, 0)
        rows = np.arange(self.tokens)
        with np.errstate(all="ignore"):
            l = self.x64 @ self.w64.T + self.b64
            m = l.max(1)
            self.lse = m + np.log(np.exp(l - m[:, None]).sum(1))
            self.loss = np.where(live, np.where(named, self.lse - l[rows, at], np.nan), 0.0)
            p = np.exp(l - self.lse[:, None])
            # scores: width additions of products, the bias; twice for what a matrix instruction does inside
            el = 2 * (self.width + 2) * U * (np.abs(self.x64) @ np.abs(self.w64).T + np.abs(self.b64))
            el = np.where(np.isfinite(l), el, 0.0)
            big = np.where(np.isfinite(l), np.abs(l), 0.0).max(1)
            # lse: the largest score error, a sum of vocab exponentials (256 in a row, then pairs and tiles of them), a
            # logarithm and roundings of numbers of the scores' size
            self.elogit = el
            self.else_ = el.max(1) + (256 + self.vocab / 64 / 16 + 40) * U * 2 + 8 * U * (big + np.abs(self.lse))
            self.eloss = self.else_ + el[rows, at] + 4 * U * (np.abs(self.lse) + big)
            g = p.copy()
            g[rows[named], at[named]] -= 1.0
            g[~live] = 0.0
            ep = p * (el + self.else_[:, None] + 8 * U * (big + np.abs(self.lse))[:, None] + 2.0 ** -22)
            ep[~live] = 0.0
        gs = self.gs.astype(np.float64) * live
        size = np.abs(gs)                                            # bounds go by the magnitude of the weights
        x = np.where(live[:, None], self.x64, 0.0)
        h = HALF[self.dtype]
        eg = ep + h * (np.abs(g) + ep) + U * np.abs(g)               # the operands' rounding
        # an exponential, its product with the weight or an operand below the smallest normal number may become 0:
        # each of the three is off by up to 2^-126 (scores far apart: exp(-87) is that small)
        eg = eg + 3 * TINY
        self.g = g
        wsafe = self.w64
        self.dx = gs[:, None] * (g @ wsafe)
        self.edx = size[:, None] * ((eg + 2 * (self.vocab + 70) * U * np.abs(g)) @ np.abs(wsafe))
        self.dw = (g * gs[:, None]).T @ x
        self.edw = ((eg + 2 * (self.tokens + 70) * U * np.abs(g)) * size[:, None]).T @ np.abs(x)
        self.db = (g * gs[:, None]).sum(0)
        self.edb = ((ep + 3 * TINY + (self.tokens + 4) * U * np.abs(g)) * size[:, None]).sum(0)
        for name in ("dx", "dw", "db"):
            value, e = getattr(self, name), getattr(self, "e" + name)
            setattr(self, "e" + name, e + h * (np.abs(value) + e) + 1e-38)
        return self

    def outputs(self, fill=float("nan")):
        self.o_loss, self.o_lse = blank((self.tokens,)), blank((self.tokens,))
        self.o_dx = blank((self.tokens, self.xs or self.width), self.dtype, fill)
        self.o_dw = blank((self.vocab, self.ws or self.width), self.dtype, fill)
        self.o_db = blank((self.vocab,), self.dtype) if self.b is not None else None

    def check_loss(self):
        near(values(self.o_lse), self.lse, self.else_)
        near(values(self.o_loss), self.loss, np.where(np.isfinite(self.eloss), self.eloss, 0))

    def check_gradients(self):
        near(values(self.o_dx)[:, :self.width], self.dx, self.edx)
        near(values(self.o_dw)[:, :self.width], self.dw, self.edw)
        if self.b is not None:
            near(values(self.o_db), self.db, self.edb)

    def forward(self, piece=0):
        drv, a = driver(), self.args(piece)
        n = drv.vocab_loss_workspace_bytes(a, training=False)
        ws = space(n)
        drv.vocab_loss_forward(self.o_loss, self.o_lse, self.x, self.w, self.b, ints(self.labels), a, ws.ptr, n)
        assert ws.intact()

    def backward(self, piece=0, gs=True):
        drv, a = driver(), self.args(piece)
        n = drv.vocab_loss_workspace_bytes(a)
        ws = space(n)
        drv.vocab_loss_backward(self.o_dx, self.o_dw, self.o_db, self.x, self.w, self.b, ints(self.labels), self.o_lse,
                                up(self.gs)[0] if gs else None, a, ws.ptr, n)
        assert ws.intact()

    def both(self, piece=0):
        drv, a = driver(), self.args(piece)
        n = drv.vocab_loss_workspace_bytes(a)
        ws = space(n)
        drv.vocab_loss_forward_backward(self.o_loss, self.o_lse, self.o_dx, self.o_dw, self.o_db, self.x, self.w, self.b,
                                        ints(self.labels), up(self.gs)[0], a, ws.ptr, n)
        assert ws.intact()


SIZES = [(1, 1, 1), (1, 64, 300), (2, 8, 257), (5, 200, 1000), (16, 100, 4000), (31, 33, 511), (33, 40, 513), (64, 256, 1024),
         (65, 72, 700), (130, 129, 259), (255, 1000, 1003), (300, 64, 2500), (1023, 96, 777)]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("tokens, width, vocab", SIZES)
def test_vocab_loss(dtype, tokens, width, vocab):
    """Forward, backward and both in one call (which keeps the scores), with and without pieces."""
    v = Vocab(dtype, tokens, width, vocab, bias=(tokens + vocab) % 2 == 0, peaked=tokens % 3 == 0).reference()
    for piece in (0, 256):
        v.outputs()
        v.forward(piece)
        v.check_loss()
        v.backward(piece)
        v.check_gradients()
        v.outputs()
        v.both(piece)
        v.check_loss()
        v.check_gradients()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 33, 64, 65])
@pytest.mark.parametrize("width, vocab, gap", [(1, 2, 0), (7, 5, 1), (119, 4099, 0), (128, 1023, 3), (130, 3, 8), (257, 70001, 0),
                                               (520, 1500, 1), (1030, 801, 5), (4096, 66, 0), (9000, 130, 0)])
def test_vocab_loss_of_a_few_tokens(dtype, tokens, width, vocab, gap):
    """The loss alone, of as few tokens as have a kernel of their own and of one more: whole and ragged rows, one to many
    sets of rows for each wave, waves that share rows, x of more than the shared memory's share."""
    v = Vocab(dtype, tokens, width, vocab, bias=(tokens + vocab) % 2 == 0, gap=gap, peaked=tokens == 15).reference()
    for piece in (0, 256):
        v.outputs()
        v.forward(piece)
        v.check_loss()
    half = vocab // 2
    if v.b is not None:                                            # masked entries leave the others as they were
        v.b[half + 1:] = float("-inf")
        v.b64 = v.b.double().cpu().numpy()
        v.labels = np.minimum(v.labels, half)
        v.reference()
        v.outputs()
        v.forward()
        v.check_loss()


@pytest.mark.parametrize("dtype, tokens, width, vocab", [("f32", 2, 2311, 16400), ("f32", 20, 1201, 33001), ("bf16", 33, 1211, 66003),
                                                         ("bf16", 64, 1155, 16385), ("f32", 64, 579, 131100)])
def test_vocab_loss_of_a_few_tokens_by_panels_of_the_width(dtype, tokens, width, vocab):
    """x of more than the shared memory's share, with rows enough that each panel is staged for more than one set of them."""
    v = Vocab(dtype, tokens, width, vocab, bias=tokens != 20).reference()
    v.outputs()
    v.forward()
    name = driver().lib.cct_hip_last_kernel().decode()
    assert name.startswith("vocab_few_kernel<") and ", true>" in name and name.endswith("rows=%d" % max(1, vocab // 65536)), name
    v.check_loss()


@pytest.mark.parametrize("dtype", BOTH)
def test_vocab_loss_of_a_few_tokens_with_scores_that_do_not_exist(dtype):
    """A fully masked vocabulary, a NaN in one token's states, a label outside: each stays with its own token."""
    v = Vocab(dtype, 4, 40, 600, bias=True, ignore=-100)
    v.labels[:] = [5, 600, 7, -100]
    v.reference()
    v.x[2, 3] = float("nan")
    v.outputs()
    v.forward()
    lse, loss = values(v.o_lse), values(v.o_loss)
    near(lse[[0, 1, 3]], v.lse[[0, 1, 3]], v.else_[[0, 1, 3]])
    near(loss[[0]], v.loss[[0]], v.eloss[[0]])
    assert np.isnan(lse[2]) and np.isnan(loss[[1, 2]]).all() and loss[3] == 0
    v.b[:] = float("-inf")
    v.outputs()
    v.forward()
    assert (values(v.o_lse)[[0, 1, 3]] == -np.inf).all() and np.isnan(values(v.o_loss)[[0, 1, 2]]).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("tokens, width, vocab, piece", [(4500, 72, 4600, 0), (2100, 520, 2300, 512), (700, 2304, 900, 0)])
def test_vocab_loss_with_the_largest_tiles(dtype, tokens, width, vocab, piece):
    """Enough rows and columns for the 256 x 256 tiles, in every use of the product."""
    v = Vocab(dtype, tokens, width, vocab, bias=True).reference()
    v.outputs()
    v.forward(piece)
    v.check_loss()
    v.backward(piece)
    v.check_gradients()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("tokens, width, vocab, piece, gap", [(1023, 520, 17011, 0, 0), (600, 300, 30011, 0, 4), (257, 520, 34011, 30000, 0)])
def test_vocab_loss_with_the_rows_past_whole_rounds_of_tiles(dtype, tokens, width, vocab, piece, gap):
    """More tiles than the chip holds at once: the last rows take another tile, in the loss, in G with its column sums
    and in dw."""
    v = Vocab(dtype, tokens, width, vocab, bias=True, gap=gap).reference()
    with tuning("vocab_keep", 2):
        v.outputs()
        v.forward(piece)
        v.check_loss()
        v.backward(piece)
        v.check_gradients()
        if gap:
            import torch
            assert bool(torch.isnan(v.o_dw[:, width:]).all()) and bool(torch.isnan(v.o_dx[:, width:]).all())


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("tokens, width, vocab", [(1, 33, 270001), (3, 2900, 17001), (100, 40, 33000), (256, 64, 16384)])
def test_vocab_loss_with_kept_scores_cut_into_ranges(dtype, bias, tokens, width, vocab):
    """Long rows of few tokens, with one part along the width and with several; labels in the first and the last range."""
    v = Vocab(dtype, tokens, width, vocab, bias=bias, peaked=tokens == 100)
    v.labels[0], v.labels[-1] = vocab - 1, min(5, vocab - 1) if tokens > 1 else vocab - 1
    v.reference()
    with tuning("vocab_keep", 1):
        v.outputs()
        v.forward()
        v.check_loss()
        v.backward()
        v.check_gradients()
        v.outputs()
        v.both()
        v.check_loss()
        v.check_gradients()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("tile", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("keep", [1, 2])
@pytest.mark.parametrize("tokens, width, vocab", [(3, 8, 5), (100, 264, 700), (333, 77, 515), (70, 1048, 1030)])
def test_vocab_loss_every_tile_with_scores_kept_or_not(dtype, tile, keep, tokens, width, vocab):
    v = Vocab(dtype, tokens, width, vocab, bias=tokens != 100).reference()
    with tuning("vocab_tile", tile), tuning("vocab_keep", keep):
        v.outputs()
        v.forward()
        v.check_loss()
        v.backward()
        v.check_gradients()
        v.outputs()
        v.both()
        v.check_loss()
        v.check_gradients()
        if keep == 2:
            v.outputs()
            v.both(piece=256)
            v.check_loss()
            v.check_gradients()


@pytest.mark.parametrize("dtype", BOTH)
def test_vocab_loss_with_strides_leaves_the_gaps_alone(dtype):
    for gap in (1, 8):
        v = Vocab(dtype, 70, 120, 300, bias=False, gap=gap).reference()
        v.outputs(fill=5.0)
        v.both()
        v.check_loss()
        v.check_gradients()
        assert (values(v.o_dx)[:, 120:] == 5.0).all() and (values(v.o_dw)[:, 120:] == 5.0).all()


@pytest.mark.parametrize("dtype", BOTH)
def test_operators_on_columns_of_wider_matrices(dtype):
    """Rows that start at an element's alignment: every matrix is a view from the second column on."""
    import torch
    from caffecontroll_amd.driver import embedding_args, vocab_loss_args
    drv, v = driver(), Vocab(dtype, 90, 77, 700, bias=True).reference()

    def view(t, fill):
        whole = torch.full((t.shape[0], t.shape[1] + 19), fill, dtype=t.dtype, device="cuda")
        whole[:, 1:1 + t.shape[1]] = t
        return whole, whole[:, 1:1 + t.shape[1]]

    (xw, x), (ww, w) = view(v.x, float("nan")), view(v.w, float("nan"))
    (dxw, dx), (dww, dw) = view(torch.zeros_like(v.x), 7.0), view(torch.zeros_like(v.w), 7.0)
    v.outputs()
    v.o_dx, v.o_dw = dx, dw
    a = vocab_loss_args(90, 77, 700, code(dtype), x_stride=96, w_stride=96)
    n = drv.vocab_loss_workspace_bytes(a)
    drv.vocab_loss_forward_backward(v.o_loss, v.o_lse, dx, dw, v.o_db, x, w, v.b, ints(v.labels), up(v.gs)[0], a,
                                    space(n).ptr, n)
    v.check_loss()
    v.check_gradients()
    for t in (dxw, dww):
        assert (t[:, 0] == 7.0).all() and (t[:, 78:] == 7.0).all()
    ids = np.random.default_rng(3).integers(0, 700, 90)
    ea = embedding_args(90, 77, 700, code(dtype), 2.0, -1, 96, 96)
    outw, out = view(torch.zeros_like(v.x), 7.0)
    drv.embedding_forward(out, w, ints(ids), ea)
    near(values(out), 2.0 * v.w64[ids], 0.0)                    # a power of two: exact
    drv.embedding_backward(dw, out, ints(ids), ea, None, 0)
    want = np.zeros((700, 77))
    np.add.at(want, ids, 2.0 * values(out))
    size = np.zeros((700, 77))
    np.add.at(size, ids, 2.0 * np.abs(values(out)))
    near(values(dw), want, (90 * U + HALF[dtype]) * size)
    for t in (outw, dww):
        assert (t[:, 0] == 7.0).all() and (t[:, 78:] == 7.0).all()


@pytest.mark.parametrize("dtype", BOTH)
def test_vocab_loss_labels_outside_the_vocabulary_and_ignored_tokens(dtype):
    import torch
    v = Vocab(dtype, 40, 64, 500, bias=True, ignore=-100)
    v.labels[3], v.labels[4], v.labels[5] = 500, -1, 2 ** 31 - 1
    v.labels[[0, 6, 7]] = -100
    v.reference()
    # what an ignored token holds stays out of everything but its own lse
    v.x[6] = float("nan")
    v.x[7] = float("inf")
    v.lse[[6, 7]] = np.nan
    for both in (False, True):
        v.outputs()
        if both:
            v.both()
        else:
            v.forward()
            v.backward()
        lse = values(v.o_lse)
        lse[[6, 7]] = np.nan
        near(lse, v.lse, v.else_)
        near(values(v.o_loss), v.loss, np.where(np.isfinite(v.eloss), v.eloss, 0))
        assert np.isnan(values(v.o_loss)[[3, 4, 5]]).all() and (values(v.o_loss)[[0, 6, 7]] == 0).all()
        v.check_gradients()
    # an ignore label that is itself an entry, and a batch of nothing but ignored tokens
    v = Vocab(dtype, 9, 16, 30, bias=False, ignore=4)
    v.labels[:] = 4
    v.reference()
    v.outputs()
    v.both()
    assert (values(v.o_loss) == 0).all() and (values(v.o_dx) == 0).all() and (values(v.o_dw) == 0).all()
    near(values(v.o_lse), v.lse, v.else_)
    assert torch.isfinite(v.o_lse).all()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("lowest", [-np.inf, -3e38])
def test_vocab_loss_masked_vocabulary(dtype, lowest):
    """A vocabulary padded to a round size: whole tiles of the bias at -inf or at the type's lowest values."""
    v = Vocab(dtype, 50, 96, 1100, bias=True)
    v.b[300:700] = lowest
    v.b[1000:] = lowest
    v.b64 = v.b.double().cpu().numpy()
    v.labels = np.where(v.labels < 0, v.labels, v.labels % 300)
    v.labels[9] = 650                                          # a label on a masked row: its loss is that large
    v.reference()
    v.else_ = np.minimum(v.else_, 1e-3)                        # (the masked rows' rounding does not reach the sum)
    for piece in (0, 256):
        v.outputs()
        v.both(piece)
        near(values(v.o_lse), v.lse, v.else_)
        got = values(v.o_loss)
        assert got[9] == np.inf if lowest == -np.inf else got[9] > 1e38
        keep = np.arange(50) != 9
        near(got[keep], v.loss[keep], 2e-3)
        assert np.isfinite(values(v.o_dx)).all() and np.isfinite(values(v.o_dw)).all()
        dw = values(v.o_dw)
        assert (dw[300:650] == 0).all() and (dw[651:700] == 0).all() and (dw[1000:] == 0).all()


def test_vocab_loss_of_a_fully_masked_row_is_nan_alone():
    """Every score -inf: the softmax of that row does not exist, the others are as they were."""
    v = Vocab("f32", 6, 4, 300, bias=False)
    v.labels[:] = np.arange(6)
    v.x64[2] = 0.0
    v.x64[2, 0] = -np.inf
    v.w64[:, 0] = np.abs(v.w64[:, 0]) + 0.1
    v.x, v.x64 = up(v.x64)
    v.w, v.w64 = up(v.w64)
    v.reference()
    v.outputs()
    v.forward()
    keep = np.arange(6) != 2
    near(values(v.o_lse)[keep], v.lse[keep], v.else_[keep])
    near(values(v.o_loss)[keep], v.loss[keep], v.eloss[keep])
    assert values(v.o_lse)[2] == -np.inf and np.isnan(values(v.o_loss)[2])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("kind", ["equal", "zero", "negative", "far apart"])
def test_vocab_loss_weights(dtype, kind):
    v = Vocab(dtype, 60, 72, 400, bias=True)
    rng = np.random.default_rng(2)
    if kind == "equal":
        v.gs[:] = 1.0 / 57
    elif kind == "zero":
        v.gs[:] = 0.0
    elif kind == "negative":
        v.gs = -v.gs
    else:
        v.gs = (10.0 ** rng.uniform(-12, 6, 60)).astype(np.float32)
    v.reference()
    for keep in (1, 2):
        with tuning("vocab_keep", keep):
            v.outputs()
            v.both()
            v.check_gradients()


@pytest.mark.parametrize("dtype", BOTH)
def test_vocab_loss_each_gradient_alone_and_without_weights(dtype):
    v = Vocab(dtype, 48, 80, 600, bias=True).reference()
    v.outputs()
    v.both()
    want = [host(t.float()).copy() for t in (v.o_dx, v.o_dw, v.o_db)]
    drv, a = driver(), v.args()
    n = drv.vocab_loss_workspace_bytes(a)
    for i, name in enumerate(("o_dx", "o_dw", "o_db")):
        v.o_dx = v.o_dw = v.o_db = None
        shape = ((48, 80), (600, 80), (600,))[i]
        setattr(v, name, blank(shape, dtype))
        drv.vocab_loss_forward_backward(v.o_loss, v.o_lse, v.o_dx, v.o_dw, v.o_db, v.x, v.w, v.b, ints(v.labels),
                                        up(v.gs)[0], a, space(n).ptr, n)
        np.testing.assert_array_equal(host(getattr(v, name).float()), want[i])
    v.gs[:] = 1.0
    v.reference()
    v.outputs()
    v.forward()
    v.backward(gs=False)
    v.check_gradients()


def test_vocab_loss_without_tokens_clears_the_weight_gradients():
    from caffecontroll_amd.driver import vocab_loss_args
    drv = driver()
    a = vocab_loss_args(0, 40, 300)
    n = drv.vocab_loss_workspace_bytes(a)
    w, _ = up(np.ones((300, 40)))
    for call in (lambda dw, db: drv.vocab_loss_backward(None, dw, db, None, w, None, None, None, None, a, space(n).ptr, n),
                 lambda dw, db: drv.vocab_loss_forward_backward(None, None, None, dw, db, None, w, None, None, None, a,
                                                                space(n).ptr, n)):
        dw, db = blank((300, 40)), blank((300,))
        call(dw, db)
        assert (host(dw) == 0).all() and (host(db) == 0).all()
    drv.vocab_loss_forward(None, None, None, None, None, None, a, None, 0)


def test_vocab_loss_gradient_against_differences():
    """Central differences of the 64-bit definition along random directions."""
    v = Vocab("f32", 12, 24, 310, bias=True).reference()
    v.outputs()
    v.both()
    rng = np.random.default_rng(8)
    live = v.labels != v.ignore

    def total(x, w, b):
        l = x @ w.T + b
        lse = np.log(np.exp(l - l.max(1)[:, None]).sum(1)) + l.max(1)
        return float((v.gs * live * np.where(live, lse - l[np.arange(12), np.where(live, v.labels, 0)], 0)).sum())

    for _ in range(4):
        d = [rng.standard_normal(a.shape) for a in (v.x64, v.w64, v.b64)]
        e = 1e-5
        diff = (total(v.x64 + e * d[0], v.w64 + e * d[1], v.b64 + e * d[2])
                - total(v.x64 - e * d[0], v.w64 - e * d[1], v.b64 - e * d[2])) / (2 * e)
        got = sum((values(o) * k).sum() for o, k in zip((v.o_dx, v.o_dw, v.o_db), d))
        bound = sum((eb * np.abs(k)).sum() for eb, k in zip((v.edx, v.edw, v.edb), d))
        # a third derivative of order 1e2 times e^2, and the cancellation of the two sums
        assert abs(got - diff) <= bound + 1e-6 * max(1.0, abs(diff))


# ---- distillation --------------------------------------------------------------------------------------------------
class Distill:
    def __init__(self, dtype, tokens, vocab, top, temperature=2.0, gap=0, seed=0):
        rng = np.random.default_rng(seed + tokens + vocab * 3 + top)
        self.dtype, self.tokens, self.vocab, self.top, self.T = dtype, tokens, vocab, top, temperature
        self.ls, self.ts = (vocab + gap if gap else 0), (top + gap if gap else 0)
        self.z, self.z64 = up(rng.standard_normal((tokens, vocab)) * 3, dtype, self.ls)
        self.ids = rng.integers(0, vocab, (tokens, top))        # the same entry may come twice
        self.ids[rng.random((tokens, top)) < 0.1] = -1
        self.tl = (rng.standard_normal((tokens, top)) * 3).astype(np.float32)
        self.gs = rng.random(tokens).astype(np.float32) + 0.1

    def upload(self):
        import torch
        self.d_tl = up(self.tl, "f32", self.ts)[0]
        ids = np.full((self.tokens, self.ts or self.top), 2 ** 31 - 1, np.int32)
        ids[:, :self.top] = self.ids
        self.d_ids = torch.from_numpy(ids).cuda()
        return self

    def args(self):
        from caffecontroll_amd.driver import distill_loss_args
        return distill_loss_args(self.tokens, self.vocab, self.top, code(self.dtype), self.T, self.ls, self.ts)

    def reference(self):
        T, n = float(np.float32(self.T)), self.tokens
        rows = np.arange(n)[:, None]
        with np.errstate(all="ignore"):
            z = self.z64 / T
            m = z.max(1)
            self.lse = m + np.log(np.exp(z - m[:, None]).sum(1))
            tau = np.where(self.ids >= 0, self.tl.astype(np.float64) / T, -np.inf)
            tm = tau.max(1)
            tm = np.where(np.isnan(tau).any(1), np.nan, tm)
            some = ~(tm == -np.inf)
            q = np.where(some[:, None], np.exp(tau - np.where(some, tm, 0)[:, None]), 0.0)
            qs = np.where(some, q.sum(1), 1.0)
            q /= qs[:, None]
            logq = tau - (tm + np.log(qs))[:, None]
            outside = self.ids >= self.vocab
            at = np.where((self.ids >= 0) & ~outside, self.ids, 0)
            term = np.where(~(q == 0), q * (logq - z[rows, at] + self.lse[:, None]), 0.0)
            self.loss = np.where(outside.any(1), np.nan, T * T * term.sum(1))
            p = np.exp(z - self.lse[:, None])
            big = np.where(np.isfinite(z), np.abs(z), 0).max(1)
            tbig = np.where(np.isfinite(tau), np.abs(tau), 0).max(1)
            # roundings of numbers of the scores' size; a lane's run of additions, pairs, ranges
            self.else_ = 12 * U * (big + np.abs(self.lse) + 1) + (self.vocab / 256 + 100) * U * 2
            eterm = 16 * U * (big + tbig + np.abs(self.lse) + 1) + self.else_
            eq = q * (12 * U * (tbig + 1) + (self.top / 64 + 10) * U * 2 + 2.0 ** -21)[:, None]
            size = np.where(q > 0, np.abs(logq - z[rows, at] + self.lse[:, None]), 0.0)
            size = np.where(np.isfinite(size), size, 0.0)
            self.eloss = T * T * ((eq * size).sum(1) + q.sum(1) * eterm + (self.top / 64 + 8) * U * (q * size).sum(1)) + 1e-30
            g = p.copy()
            ok = ~(q == 0) & (self.ids >= 0) & ~outside
            for t in range(n):
                np.subtract.at(g[t], at[t][ok[t]], q[t][ok[t]])
            g[~some] = 0.0
            eqs = np.zeros_like(g)
            for t in range(n):
                np.add.at(eqs[t], at[t][ok[t]], eq[t][ok[t]] + self.top * U * q[t][ok[t]])
            w = T * self.gs.astype(np.float64)
            self.d = w[:, None] * g
            e = w[:, None] * (p * (self.else_ + 12 * U * (big + np.abs(self.lse)) + 2.0 ** -21)[:, None] + eqs + 4 * U * np.abs(g))
            e[~some] = 0.0
            self.ed = e + HALF[self.dtype] * (np.abs(self.d) + e) + 1e-38
        return self

    def outputs(self):
        self.o_loss, self.o_lse = blank((self.tokens,)), blank((self.tokens,))
        self.o_d = blank((self.tokens, self.ls or self.vocab), self.dtype, 5.0)

    def check(self, gradient=True):
        near(values(self.o_lse), self.lse, self.else_)
        near(values(self.o_loss), self.loss, np.where(np.isfinite(self.eloss), self.eloss, 0))
        if gradient:
            near(values(self.o_d)[:, :self.vocab], self.d, self.ed)
            assert (values(self.o_d)[:, self.vocab:] == 5.0).all()

    def run(self, both, in_place=False, gs=True):
        drv, a = driver(), self.args()
        n = drv.distill_loss_workspace_bytes(a)
        ws = space(n)
        self.outputs()
        z, d = self.z, self.o_d
        if in_place:
            z = self.z.clone()
            if self.ls:
                z[:, self.vocab:] = 5.0
            d = self.o_d = z
        g = up(self.gs)[0] if gs else None
        if both:
            drv.distill_loss_forward_backward(self.o_loss, self.o_lse, d, z, self.d_ids, self.d_tl, g, a, ws.ptr, n)
        else:
            drv.distill_loss_forward(self.o_loss, self.o_lse, z, self.d_ids, self.d_tl, a, ws.ptr, n)
            drv.distill_loss_backward(d, z, self.d_ids, self.d_tl, self.o_lse, g, a, ws.ptr, n)
        assert ws.intact()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("tokens, vocab, top, gap", [
    (1, 1, 1, 0), (1, 7, 3, 0), (1, 50021, 100, 0), (2, 131072, 8, 0), (3, 9000, 1, 3), (32, 1000, 10, 0), (100, 257, 64, 0),
    (65, 4097, 1024, 8), (300, 5000, 65, 1), (7, 65536, 33, 0), (5, 70001, 20, 0), (2, 140000, 5, 0), (600, 33000, 4, 0)])
def test_distill_loss(dtype, tokens, vocab, top, gap):
    d = Distill(dtype, tokens, vocab, top, gap=gap).upload().reference()
    for both in (False, True):
        for in_place in (False, True):
            d.run(both, in_place)
            d.check()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("vocab", [300, 9001])
def test_distill_loss_lists_that_are_empty_masked_or_wrong(dtype, vocab):
    d = Distill(dtype, 12, vocab, 20, temperature=0.7)
    d.ids[0] = -1                                               # no list at all
    d.tl[1] = -np.inf                                           # no entry with weight
    d.ids[2, :] = 5                                             # one entry, many times
    d.ids[3, 4] = vocab                                         # a row that does not exist
    d.ids[4, 1:] = -1
    d.ids[4, 0] = vocab - 1                                     # a single entry
    d.tl[5, ::2] = -np.inf
    d.tl[6] = -3.4e38                                           # the type's lowest values, all alike
    d.tl[7, 3] = 500.0                                          # one entry far above the rest
    d.tl[0, 3] = np.nan                                         # in an absent entry
    d.ids[11, 1:], d.ids[11, 0], d.tl[11, 0] = -1, 3, np.nan    # nothing but a NaN: so is the token's loss
    d.z[8, 10:200] = float("-inf")                              # a masked vocabulary, the list elsewhere
    d.ids[8] = 250
    d.z[9, :] = float("-inf")
    d.z[9, 7] = 1.0
    d.ids[9] = 7
    d.z[10, 100] = float("-inf")
    d.ids[10, 0], d.tl[10, 0] = 100, 1.0                        # weight where the student has none: an infinite loss
    d.z64 = d.z.double().cpu().numpy()
    d.upload().reference()
    assert d.loss[10] == np.inf and np.isnan(d.loss[[3, 11]]).all() and (d.loss[:2] == 0).all()
    d.ed = np.where(np.isnan(d.ed), 0.0, d.ed)
    for both in (False, True):
        d.run(both)
        d.check()
        assert (values(d.o_d)[:2] == 0).all() and (values(d.o_loss)[:2] == 0).all()


def test_distill_loss_without_weights_and_gradient_against_differences():
    d = Distill("f32", 6, 400, 12, temperature=1.5)
    d.gs[:] = 1.0
    d.upload().reference()
    d.run(True, gs=False)
    d.check()
    rng = np.random.default_rng(4)
    base = d.z64
    got = values(d.o_d)
    for _ in range(3):
        k, e = rng.standard_normal(base.shape), 1e-5
        sums = []
        for s in (1, -1):
            d.z64 = base + s * e * k
            sums.append(d.reference().loss.sum())
        d.z64 = base
        d.reference()
        diff = (sums[0] - sums[1]) / (2 * e)
        assert abs((got * k).sum() - diff) <= (d.ed * np.abs(k)).sum() + 1e-6 * max(1.0, abs(diff))


def test_distill_loss_without_tokens():
    from caffecontroll_amd.driver import distill_loss_args
    drv, a = driver(), distill_loss_args(0, 10, 3)
    drv.distill_loss_forward(None, None, None, None, None, a, None, 0)
    drv.distill_loss_backward(None, None, None, None, None, None, a, None, 0)
    drv.distill_loss_forward_backward(None, None, None, None, None, None, None, a, None, 0)
