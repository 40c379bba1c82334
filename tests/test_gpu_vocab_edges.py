"""The vocabulary operators where values are not finite, near the type's limits or cancel, against their definitions in 64
bits with the bounds of test_gpu_vocab_ops."""
import numpy as np
import pytest

from gpu_util import tuning
from test_gpu_vocab_ops import BOTH, Vocab, near, values

pytestmark = pytest.mark.gpu


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
