"""What the embedding, vocabulary loss and distillation entry points refuse: checked before the device is touched, so
these run anywhere."""
import ctypes as C

import pytest

from caffecontroll_amd import CctHipError, _lib
from caffecontroll_amd.driver import BF16, F32, HIPDriver, distill_loss_args, embedding_args, vocab_loss_args

A = 1 << 20  # an address that is never followed


@pytest.fixture()
def drv():
    d = HIPDriver.__new__(HIPDriver)   # no device is selected
    d.lib = _lib.load()
    return d


def refused(call, *args, match, **kw):
    with pytest.raises(CctHipError, match=match) as e:
        call(*args, **kw)
    assert "code 100001" in str(e.value)


def test_argument_blocks_have_the_header_s_layout():
    assert C.sizeof(_lib.EmbeddingArgs) == 40 and _lib.EmbeddingArgs.table_stride.offset == 24
    assert C.sizeof(_lib.VocabLossArgs) == 40 and _lib.VocabLossArgs.x_stride.offset == 24
    assert C.sizeof(_lib.DistillLossArgs) == 40 and _lib.DistillLossArgs.logits_stride.offset == 24


@pytest.mark.parametrize("bad, match", [
    (dict(tokens=-1), "tokens -1"), (dict(width=0), "width 0"), (dict(vocab=0), "vocab 0"), (dict(dtype=2), "dtype 2"),
    (dict(dtype=-1), "dtype -1"), (dict(table_stride=7), "stride"), (dict(out_stride=1), "stride"),
    (dict(tokens=(1 << 23) + 1), "at most"), (dict(vocab=(1 << 26) + 1), "at most"), (dict(width=(1 << 20) + 1), "at most"),
])
def test_embedding_refuses(drv, bad, match):
    a = embedding_args(**{**dict(tokens=4, width=8, vocab=10), **bad})
    refused(drv.embedding_forward, A, A, A, a, match=match)
    refused(drv.embedding_backward, A, A, A, a, A, 1 << 30, match=match)
    assert drv.embedding_workspace_bytes(a) == 0


def test_embedding_refuses_arrays_and_workspaces(drv):
    a = embedding_args(1000, 8, 10, BF16)
    need = drv.embedding_workspace_bytes(a)
    assert need > 0 == drv.embedding_workspace_bytes(embedding_args(100, 8, 10, BF16))   # few tokens need none
    for i in range(3):
        arrays = [A, A, A]
        arrays[i] = None
        refused(drv.embedding_forward, *arrays, a, match="null array")
        refused(drv.embedding_backward, *arrays, a, A, need, match="null array")
    refused(drv.embedding_backward, A, A, A, a, A, need - 1, match="workspace")
    refused(drv.embedding_backward, A, A, A, a, None, need, match="workspace")
    refused(drv.embedding_backward, A, A, A, a, A + 8, need, match="workspace")
    refused(lambda: _lib.check(drv.lib.cct_hip_embedding_forward(A, A, A, None)), match="null argument block")


@pytest.mark.parametrize("bad, match", [
    (dict(tokens=-1), "tokens -1"), (dict(width=0), "width 0"), (dict(vocab=-3), "vocab -3"), (dict(dtype=7), "dtype 7"),
    (dict(piece=-1), "piece -1"), (dict(x_stride=7), "stride"), (dict(w_stride=5), "stride"),
    (dict(tokens=(1 << 20) + 1), "at most"), (dict(vocab=1 << 24), "at most"), (dict(width=(1 << 16) + 1), "at most"),
    (dict(x_stride=(1 << 20) + 1), "strides of at most"), (dict(w_stride=1 << 21), "strides of at most"),
])
def test_vocab_loss_refuses(drv, bad, match):
    a = vocab_loss_args(**{**dict(tokens=4, width=8, vocab=10), **bad})
    refused(drv.vocab_loss_forward, A, A, A, A, None, A, a, A, 1 << 40, match=match)
    refused(drv.vocab_loss_backward, A, A, None, A, A, None, A, A, None, a, A, 1 << 40, match=match)
    refused(drv.vocab_loss_forward_backward, A, A, A, A, None, A, A, None, A, None, a, A, 1 << 40, match=match)
    assert drv.vocab_loss_workspace_bytes(a) == 0


def test_vocab_loss_refuses_arrays_and_workspaces(drv):
    a = vocab_loss_args(100, 8, 1000, F32)
    need, forward = drv.vocab_loss_workspace_bytes(a), drv.vocab_loss_workspace_bytes(a, training=False)
    assert 0 < forward < need
    for i in (0, 1, 2, 3, 5):
        arrays = [A, A, A, A, None, A]
        arrays[i] = None
        refused(drv.vocab_loss_forward, *arrays, a, A, forward, match="null array")
    for i in (3, 4, 6, 7):
        arrays = [A, A, None, A, A, None, A, A, None]
        arrays[i] = None
        refused(drv.vocab_loss_backward, *arrays, a, A, need, match="null array")
    for i in (0, 1, 5, 6, 8):
        arrays = [A, A, A, A, None, A, A, None, A, None]
        arrays[i] = None
        refused(drv.vocab_loss_forward_backward, *arrays, a, A, need, match="null array")
    refused(drv.vocab_loss_backward, None, None, None, A, A, None, A, A, None, a, A, need, match="no gradient")
    refused(drv.vocab_loss_forward_backward, A, A, None, None, None, A, A, None, A, None, a, A, need, match="no gradient")
    refused(drv.vocab_loss_forward, A, A, A, A, None, A, a, A, forward - 1, match="workspace")
    refused(drv.vocab_loss_forward, A, A, A, A, None, A, a, A + 4, forward, match="workspace")
    refused(drv.vocab_loss_backward, A, A, None, A, A, None, A, A, None, a, A, forward, match="workspace")
    refused(drv.vocab_loss_forward_backward, A, A, A, A, None, A, A, None, A, None, a, None, need, match="workspace")


def test_vocab_loss_refuses_rows_of_whole_chunks_that_start_between_them(drv):
    for dtype, width, off in ((BF16, 8, 2), (F32, 4, 4), (BF16, 64, 8)):
        a = vocab_loss_args(10, width, 300, dtype)
        n = drv.vocab_loss_workspace_bytes(a)
        for x, w in ((A + off, A), (A, A + off)):
            refused(drv.vocab_loss_forward, A, A, x, w, None, A, a, A, n, match="multiple of 16")
            refused(drv.vocab_loss_backward, A, A, None, x, w, None, A, A, None, a, A, n, match="multiple of 16")
            refused(drv.vocab_loss_forward_backward, A, A, A, A, None, x, w, None, A, None, a, A, n, match="multiple of 16")


def test_vocab_loss_workspace_stays_bounded():
    """The workspace goes by tokens and piece, not by tokens * vocab; pieces smaller than the automatic ones need less."""
    d = HIPDriver.__new__(HIPDriver)
    d.lib = _lib.load()
    small, large = (d.vocab_loss_workspace_bytes(vocab_loss_args(8192, 4096, v, BF16)) for v in (131072, 4 * 131072))
    # what grows with the vocabulary alone are the tiles' statistics, 8 bytes per token and tile of 64 rows or more
    assert large - small <= 3 * 131072 // 64 * 8192 * 8
    assert small < 2 << 30 < 8192 * 131072 * 4
    pieces = [d.vocab_loss_workspace_bytes(vocab_loss_args(8192, 4096, 131072, BF16, piece=p)) for p in (256, 1024, 4096)]
    assert max(pieces) < small


@pytest.mark.parametrize("bad, match", [
    (dict(tokens=-2), "tokens -2"), (dict(vocab=0), "vocab 0"), (dict(top=0), "top 0"), (dict(top=1025), "above 1024"),
    (dict(dtype=3), "dtype 3"), (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
    (dict(logits_stride=9), "stride"), (dict(top_stride=2), "stride"), (dict(tokens=(1 << 20) + 1), "at most"),
])
def test_distill_loss_refuses(drv, bad, match):
    a = distill_loss_args(**{**dict(tokens=4, vocab=10, top=3), **bad})
    refused(drv.distill_loss_forward, A, A, A, A, A, a, A, 1 << 30, match=match)
    refused(drv.distill_loss_backward, A, A, A, A, A, None, a, A, 1 << 30, match=match)
    refused(drv.distill_loss_forward_backward, A, A, A, A, A, A, None, a, A, 1 << 30, match=match)
    assert drv.distill_loss_workspace_bytes(a) == 0


def test_distill_loss_refuses_arrays_and_workspaces(drv):
    a = distill_loss_args(4, 1000, 3, BF16, temperature=2.0)
    need = drv.distill_loss_workspace_bytes(a)
    assert need > 0
    for i in range(5):
        arrays = [A] * 5
        arrays[i] = None
        refused(drv.distill_loss_forward, *arrays, a, A, need, match="null array")
        refused(drv.distill_loss_backward, *arrays, None, a, A, need, match="null array")
    for i in range(6):
        arrays = [A] * 6
        arrays[i] = None
        refused(drv.distill_loss_forward_backward, *arrays, None, a, A, need, match="null array")
    for call, n in ((drv.distill_loss_forward, 5), (drv.distill_loss_backward, 5), (drv.distill_loss_forward_backward, 6)):
        extra = [] if call == drv.distill_loss_forward else [None]
        refused(call, *[A] * n, *extra, a, A, need - 1, match="workspace")
        refused(call, *[A] * n, *extra, a, A + 2, need, match="workspace")


@pytest.mark.parametrize("temperature", [1e-45, 1e-39, 2.0 ** -61, 2.0 ** 61, 3e38])
def test_distill_loss_refuses_temperatures_whose_square_or_inverse_is_no_normal_number(drv, temperature):
    a = distill_loss_args(tokens=4, vocab=10, top=3, temperature=temperature)
    refused(drv.distill_loss_forward, A, A, A, A, A, a, A, 1 << 30, match="temperature")
    refused(drv.distill_loss_backward, A, A, A, A, A, None, a, A, 1 << 30, match="temperature")
    refused(drv.distill_loss_forward_backward, A, A, A, A, A, A, None, a, A, 1 << 30, match="temperature")
    assert drv.distill_loss_workspace_bytes(a) == 0
    for least in (2.0 ** -60, 2.0 ** 60):
        assert drv.distill_loss_workspace_bytes(distill_loss_args(4, 10, 3, temperature=least)) > 0
