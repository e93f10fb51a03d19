"""What the tests of beam selection on the GPU take for granted (CPU-only): that
their inputs leave the order of what is kept to the scores, not to roundings."""
import numpy as np
import pytest

import beam_plain as B
import decoder_plain as R
import test_gpu_beam as T
from ppocr_native_amd import decoder as D

# A score is off by its beam's logarithm of a sum of f32 exponentials, 16 steps at most: two beams' candidates change
# places only where their scores are nearer than twice that. One input has two at 2.3 steps: 700 exponentials, whose
# sums are off by less than one (half a step for each of some 10 additions in a row, of either sign).
APART = 2 * 16 * R.STEP
NEAR = {(D.F16, 1, 128, 700, 128): 2 * R.STEP}


class Inputs:
    """A call's inputs; its answer is the one in 64 bits, and is looked at instead of the GPU's."""

    nearest = np.inf

    def __init__(self, x, base, keep, t, ended=None, end=-1, gap=0):
        self.x, self.base = R.values(R.stored(x, t), t), np.asarray(base, np.float32).astype(np.float64)
        self.keep, self.ended, self.end = keep, ended, end

    def run(self, stream=0):
        pass

    def check(self):
        out = []
        for b in range(len(self.x)):
            ended = None if self.ended is None else self.ended[b]
            more, _ = B.choose(self.x[b], self.base[b], self.keep + 1, ended, self.end)
            near, parents = more[0][more[2] >= 0], more[1][more[2] >= 0]
            gaps = -np.diff(near)
            # (Within a beam the order is the logits'.)
            gaps = gaps[(parents[1:] != parents[:-1]) & (gaps > 0)]
            if len(gaps):
                Inputs.nearest = min(Inputs.nearest, gaps.min())
            out.append([o[:-1] for o in more])
        return [np.stack([o[j] for o in out]) for j in range(4)]


CALLS = [(T.test_select, dict(t=t, batch=a, beams=b, vocab=c, keep=d)) for t in R.REAL for a, b, c, d in T.SIZES]
CALLS += [(T.test_select_ties, dict(t=t)) for t in R.REAL]
CALLS += [(T.test_select_of_sorted_logits, dict(t=t, keep=k)) for t in R.REAL for k in (1, 8, 128)]
CALLS += [(T.test_select_of_what_is_not_finite, dict(t=t)) for t in R.REAL]
CALLS += [(T.test_select_among_many_equal_choices, {})]


@pytest.mark.parametrize("test,args", CALLS)
def test_scores_of_beams_are_apart(monkeypatch, test, args):
    monkeypatch.setattr(T, "Select", Inputs)
    monkeypatch.setattr(T, "synchronize", lambda: None)
    monkeypatch.setattr(Inputs, "nearest", np.inf)
    test(**args)
    assert Inputs.nearest > NEAR.get(tuple(args.values()), APART), Inputs.nearest / R.STEP
