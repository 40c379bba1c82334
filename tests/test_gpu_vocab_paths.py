"""Paths of the vocabulary operators that only some sizes and strides take, each shown to be taken by the launch record, against
the definitions in 64 bits with the bounds of test_gpu_vocab_ops."""
import re

import numpy as np
import pytest

from gpu_util import driver, tuning
from test_gpu_vocab_ops import BOTH, HALF, U, Distill, Vocab, blank, code, ints, near, space, up, values

pytestmark = pytest.mark.gpu


def last_product():
    """Tile, use, m and n of the last product that a call enqueued."""
    name = driver().lib.cct_hip_last_kernel().decode()
    m = re.match(r"vocab_product_kernel<\w+, Shape<(\d+), (\d+), [\d, ]+>, (\d), \w+, \w+> splits=\d+ m=(\d+) n=(\d+)$", name)
    assert m, name
    bm, bn, use, rows, cols = map(int, m.groups())
    return (bm, bn), use, rows, cols


class Alone:
    """Gradients asked for one at a time, so that each one's products are the last of its call."""

    def __init__(self, v, piece=0):
        self.v, self.piece, self.outputs = v, piece, (v.o_dx, v.o_dw, v.o_db)

    def run(self, name):
        v = self.v
        v.o_dx = v.o_dw = v.o_db = None
        setattr(v, name, self.outputs[("o_dx", "o_dw", "o_db").index(name)])
        v.backward(self.piece)
        v.o_dx, v.o_dw, v.o_db = self.outputs
        return last_product()


# ---- vocabulary loss -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, tokens, width, vocab, last, cut", [
    ("bf16", 839, 895, 38627, 38627, ("loss", "o_db", "o_dw")), ("bf16", 347, 712, 45383, 45383, ("loss", "o_db", "o_dw")),
    ("bf16", 33, 1008, 49742, 49742, ("o_dw",)), ("f32", 11, 3790, 10835, 10835, ("o_dw",)),
    ("f32", 1211, 23, 83088, 83088 - 65536, ("loss", "o_db"))])
def test_vocab_loss_with_a_second_launch_for_the_last_rows(dtype, tokens, width, vocab, last, cut):
    """The rows past whole rounds of tiles take another tile in a launch of their own: the loss, G with its column sums, dw; with
    all of the vocabulary in one piece, and in the `last` rows of several."""
    v = Vocab(dtype, tokens, width, vocab, bias=True)
    v.labels[0], v.labels[1] = vocab - 1, vocab - 30                # labels among those rows
    v.reference()
    with tuning("vocab_keep", 2):
        v.outputs()
        v.forward()
        _, use, rows, _ = last_product()
        assert use == 0 and (rows < last) == ("loss" in cut)
        v.check_loss()
        alone = Alone(v)
        _, use, rows, _ = alone.run("o_db")
        assert use == 1 and (rows < last) == ("o_db" in cut)
        _, use, _, rows = alone.run("o_dw")
        assert use == 3 and (rows < last) == ("o_dw" in cut)
        alone.run("o_dx")
        v.check_gradients()
        v.outputs()
        v.both()
        v.check_loss()
        v.check_gradients()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("keep, piece", [(1, 0), (2, 0), (2, 512)])
@pytest.mark.parametrize("tokens, width, vocab", [(600, 520, 2600), (300, 2312, 700)])
def test_vocab_loss_with_tiles_of_256_in_several_bands(dtype, keep, piece, tokens, width, vocab):
    """More than eight tiles of 256 x 256 along the vocabulary or the width, several along the tokens, in every use of the product."""
    v = Vocab(dtype, tokens, width, vocab, bias=True).reference()
    with tuning("vocab_tile", 1), tuning("vocab_keep", keep):
        v.outputs()
        v.forward(piece)
        tile, use, rows, cols = last_product()
        assert tile == (256, 256) and use == (2 if keep == 1 else 0) and cols == tokens
        v.check_loss()
        alone = Alone(v, piece)
        uses = [alone.run(name) for name in ("o_db", "o_dw", "o_dx")]
        assert all(u[0] == (256, 256) for u in uses) and [u[1] for u in uses[:2]] == [2 if keep == 1 else 1, 3]
        assert uses[2][1] in (2, 3) and uses[2][2:] == (width, tokens)
        v.check_gradients()
        v.outputs()
        v.both(piece)
        v.check_loss()
        v.check_gradients()


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("keep", [0, 1, 2])
@pytest.mark.parametrize("x_gap, w_gap", [(0, 3), (3, 0), (8, 3), (3, 8)])
def test_vocab_loss_with_one_operand_packed(dtype, keep, x_gap, w_gap):
    """Rows of whole 16-byte chunks in one of x and w, read as they lie, beside rows that are copied first."""
    v = Vocab(dtype, 130, 128, 1111, bias=True)
    v.xs, v.ws = (128 + g if g else 0 for g in (x_gap, w_gap))
    v.x, _ = up(v.x64, dtype, v.xs)
    v.w, _ = up(v.w64, dtype, v.ws)
    v.reference()
    with tuning("vocab_keep", keep):
        for piece in (0, 256):
            v.outputs(fill=5.0)
            v.forward(piece)
            v.check_loss()
            v.backward(piece)
            v.check_gradients()
            v.outputs(fill=5.0)
            v.both(piece)
            v.check_loss()
            v.check_gradients()
            assert (values(v.o_dx)[:, 128:] == 5.0).all() and (values(v.o_dw)[:, 128:] == 5.0).all()


def test_vocab_loss_gradients_in_pieces_past_four_gib():
    """A matrix of 2.3e9 elements in pieces of 65536 rows, one of which begins at 4 GiB: scores computed twice, dx added up
    over the pieces, and dw on both sides of that boundary."""
    import torch
    from caffecontroll_amd.driver import BF16, vocab_loss_args
    drv, vocab, width, tokens, piece = driver(), 565000, 4096, 24, 65536
    edge = 8 * piece                                               # bf16: 4 GiB from the start
    rows = torch.cat([torch.arange(edge - 32, edge + 32), torch.arange(vocab - 64, vocab)]).cuda()
    gen = torch.Generator(device="cuda").manual_seed(11)
    w = torch.zeros((vocab, width), dtype=torch.bfloat16, device="cuda")
    x = torch.randn(tokens, width, generator=gen, device="cuda").to(torch.bfloat16)
    some = (torch.randn(len(rows), width, generator=gen, device="cuda") / 16).to(torch.bfloat16)
    w[rows] = some
    at = torch.arange(tokens, device="cuda") * 5                   # places in `rows`: labels on both sides, and in the last rows
    labels = rows[at].to(torch.int32)
    a = vocab_loss_args(tokens, width, vocab, BF16, piece=piece)
    n = drv.vocab_loss_workspace_bytes(a)
    ws = space(n)
    loss, lse, db = blank((tokens,)), blank((tokens,)), blank((vocab,), "bf16")
    dx, dw = blank((tokens, width), "bf16"), blank((vocab, width), "bf16")
    bias = torch.zeros(vocab, dtype=torch.bfloat16, device="cuda")
    drv.vocab_loss_forward_backward(loss, lse, dx, None, db, x, w, bias, labels, None, a, ws.ptr, n)
    _, use, _, _ = last_product()
    assert use == 2 and ws.intact()                                # dx in parts that are added up
    drv.vocab_loss_forward_backward(loss, lse, dx, dw, db, x, w, bias, labels, None, a, ws.ptr, n)
    assert last_product()[3] <= vocab - 8 * piece and ws.intact()  # the last piece's rows
    x64, w64 = x.double(), some.double()
    s = x64 @ w64.T
    total = torch.exp(s).sum(1) + (vocab - len(rows))
    want = torch.log(total)
    # scores of a few hundred: 4096 terms of a fp32 sum, 4096 * 2^-24 of the terms' size
    size = 2.5e-4 * (x64.abs() @ w64.abs().T).amax(1)
    near(values(lse), values(want), values(size))
    near(values(loss), values(want - s[torch.arange(tokens), at]), 2 * values(size))
    g = torch.exp(s - want[:, None])
    g[torch.arange(tokens), at] -= 1.0
    rest = 1.0 / total                                             # G of every row that is zero
    # G: the scores' and lse's error, a rounding to bf16 of each entry and of the result
    eg = g.abs() * (2 * size[:, None] + 2.0 ** -8) + (g + 1).abs() * 2 * size[:, None]
    erest = rest * (2 * size + 2.0 ** -8)
    wdx = g @ w64
    edx = eg @ w64.abs()
    near(values(dx), values(wdx), values(edx + 2.0 ** -8 * (wdx.abs() + edx)) + 1e-30)
    wdw, edw = g.T @ x64, eg.T @ x64.abs()
    near(values(dw[rows]), values(wdw), values(edw + 2.0 ** -8 * (wdw.abs() + edw)) + 1e-30)
    wz, ez = rest @ x64, erest @ x64.abs()
    ez = ez + 2.0 ** -8 * (wz.abs() + ez) + 1e-30
    for r in (0, piece - 1, piece, edge - 33, edge + 32, edge + piece // 2, vocab - 65):
        near(values(dw[r]), values(wz), values(ez))
    for p in range(0, vocab, piece):                               # every row that is zero has the same gradient
        part = dw[p:p + piece]
        other = (part != dw[0]).any(1).nonzero()[:, 0] + p
        assert set(other.tolist()) <= set(rows.tolist())
    wdb, edb = g.sum(0), eg.sum(0)
    near(values(db[rows]), values(wdb), values(edb + 2.0 ** -8 * (wdb.abs() + edb)))
    assert float(db[7]) == float(db[edge + 100]) == float(db[vocab - 100])


@pytest.mark.parametrize("tokens, width, vocab, top", [(347, 712, 45383, 5), (33, 1008, 49742, 3)])
def test_calls_with_a_second_launch_in_a_replayed_graph(tokens, width, vocab, top):
    from test_gpu_vocab_model import test_every_call_in_a_replayed_graph as replay
    with tuning("vocab_keep", 2):
        replay(tokens, width, vocab, top)


# ---- distillation ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("tokens, vocab, top", [(5, 9, 2), (40, 300, 20), (3, 9001, 300), (2, 65536, 7), (3, 140000, 5)])
def test_distill_loss_on_columns_of_wider_matrices(dtype, tokens, vocab, top):
    """Rows that start at an element's alignment: the scores, their gradient and both lists are views from the second column on."""
    import torch
    from caffecontroll_amd.driver import distill_loss_args
    drv, d = driver(), Distill(dtype, tokens, vocab, top).upload().reference()

    def view(t, gap, fill):
        whole = torch.full((t.shape[0], t.shape[1] + gap), fill, dtype=t.dtype, device="cuda")
        whole[:, 1:1 + t.shape[1]] = t
        return whole, whole[:, 1:1 + t.shape[1]]

    _, z = view(d.z, 6, float("nan"))
    _, ids = view(d.d_ids, 4, 2 ** 31 - 1)
    _, tl = view(d.d_tl, 4, float("nan"))
    a = distill_loss_args(tokens, vocab, top, code(dtype), d.T, vocab + 6, top + 4)
    n = drv.distill_loss_workspace_bytes(a)
    gs = up(d.gs)[0]
    for both in (False, True):
        for in_place in (False, True):
            ws = space(n)
            d.outputs()
            dw, dz = view(z if in_place else torch.zeros_like(d.z), 6, 5.0)
            source = dz if in_place else z
            if both:
                drv.distill_loss_forward_backward(d.o_loss, d.o_lse, dz, source, ids, tl, gs, a, ws.ptr, n)
            else:
                drv.distill_loss_forward(d.o_loss, d.o_lse, source, ids, tl, a, ws.ptr, n)
                drv.distill_loss_backward(dz, source, ids, tl, d.o_lse, gs, a, ws.ptr, n)
            d.o_d = dz
            d.check()
            assert (dw[:, 0] == 5.0).all() and (dw[:, vocab + 1:] == 5.0).all() and ws.intact()


# ---- embedding -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, width", [("f32", 1029), ("bf16", 2051), ("f32", 1023), ("bf16", 2047)])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("tokens, vocab, kind, gap", [(8200, 700, "skewed", 0), (9001, 16500, "uniform", 3), (8193, 33, "one", 0),
                                                      (8300, 16700, "uniform", 0)])
def test_embedding_gradient_by_rows_and_by_tokens(dtype, width, accumulate, tokens, vocab, kind, gap):
    """Every row's tokens looked up (rows of 4 KB and more, more tokens than half the rows), or the rows with tokens visited."""
    from caffecontroll_amd.driver import embedding_args
    drv, rng = driver(), np.random.default_rng(tokens + width)
    stride = width + gap if gap else 0
    ids = {"skewed": np.minimum(rng.zipf(1.3, tokens) - 1, vocab - 1), "uniform": rng.integers(0, vocab, tokens),
           "one": np.full(tokens, vocab - 1)}[kind]
    if kind != "one":
        ids[[5, 50, 60]] = -1, vocab, -7
    dout, d64 = up(rng.standard_normal((tokens, width)), dtype, stride)
    table, old = up(rng.standard_normal((vocab, width)), dtype, stride, 3.0)
    args = embedding_args(tokens, width, vocab, code(dtype), 0.3, -1, stride, stride)
    n = drv.embedding_workspace_bytes(args)
    ws = space(n)
    drv.embedding_backward(table, dout, ints(ids), args, ws.ptr, n, accumulate)
    by_rows = width > 1024 + 1024 * (dtype == "bf16") and tokens > vocab // 2
    assert drv.lib.cct_hip_last_kernel().decode().startswith("embedding_sum_kernel<" if by_rows else "embedding_runs_kernel<")
    got = values(table)
    assert ws.intact() and (got[:, width:] == 3.0).all()
    ok = (ids >= 0) & (ids < vocab)
    count = np.bincount(ids[ok], minlength=vocab)
    order = np.argsort(ids[ok], kind="stable")
    begin = np.concatenate([[0], np.cumsum(count)[:-1]])
    some = count > 0
    total, size = np.zeros((vocab, width)), np.zeros((vocab, width))
    total[some] = np.add.reduceat(d64[ok][order], begin[some])
    size[some] = np.add.reduceat(np.abs(d64[ok][order]), begin[some])
    s32 = float(np.float32(0.3))
    want = s32 * total + (old if accumulate else 0.0)
    # count additions, the product with the scale, the addition to what was there, the rounding to the type
    bound = s32 * (count[:, None] + 1) * U * size * (1 + 1e-3) + (U * np.abs(want) if accumulate else 0)
    near(got[:, :width], want, bound + HALF[dtype] * (np.abs(want) + bound))
    if accumulate:
        assert (got[:, :width][~some] == old[~some]).all()
