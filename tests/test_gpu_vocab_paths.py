"""Paths of the vocabulary operators that only some sizes and strides take, each shown to be taken by the launch record, against
the definitions in 64 bits with the bounds of test_gpu_vocab_ops."""
import re

import numpy as np
import pytest

from gpu_util import driver, tuning
from test_gpu_vocab_ops import BOTH, Distill, Vocab, blank, ints, near, space, up, values

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
