"""The fine-tuning operators at the edges of their ranges: each test here failed before what it names was put right."""
import math

import numpy as np
import pytest
import torch

import train_ref as R
from granite_conv_b200 import training as tr
from test_gpu_training import BF, DEV, E, EPS, F32, HF, check_ctc, close, ctc_case, lens_of, rand, rng_of, rounded

pytestmark = pytest.mark.gpu


# ---- CTC: states that the logits favour in another order than the transcript -------------------------------------------
def run_case(S, at, runs, tail=40):
    """A transcript whose labels at - 1, at and at + 1 are c, a and b of classes of their own, its places in the middle
    of the frames; `runs` of (class, frames, boost) are favoured there, everything else is noise."""
    names = {"blank": 0, "a": 1, "b": 2, "c": 3}
    V = 13
    g = np.random.default_rng(S + at)
    labels = 4 + (np.arange(S) % (V - 4))
    labels[at - 1:at + 2] = (3, 1, 2)
    head = 2 * at + 4
    T = head + sum(r[1] for r in runs) + 2 * (S - at) + tail
    x = g.normal(size=(1, T, V))
    t = head
    for name, n, boost in runs:
        x[0, t:t + n, names[name]] += boost
        t += n
    return (torch.tensor(x, dtype=F32, device=DEV), torch.tensor(labels[None], dtype=torch.int32, device=DEV),
            torch.tensor([T], dtype=torch.int32, device=DEV), torch.tensor([S], dtype=torch.int32, device=DEV))


def backwards(logits, targets, il, tl):
    """The same case with frames and labels reversed: its states are those of the chain from the end."""
    return logits.flip(1).contiguous(), targets.flip(1).contiguous(), il, tl


@pytest.mark.parametrize("S,at,boost,K", [(100, 44, 16.0, 59), (200, 90, 18.0, 55), (300, 60, 12.0, 79),
                                          (300, 150, 14.0, 75), (500, 100, 10.0, 100), (500, 100, 14.0, 75)])
def test_ctc_path_from_a_lane_far_below(S, at, boost, K):
    """b, favoured first, lifts the lane of a and b more than 1000 octaves above the lane of c.  The path that counts
    waits before c through that, goes from c to a and then has a's frames: all of Z crosses between the two lanes."""
    case = run_case(S, at, [("b", K, boost), ("c", 12, boost), ("a", K + 12, boost)])
    for logits, targets, il, tl in (case, backwards(*case)):
        ref, _ = R.ctc(logits, targets, il, tl, 0, False)
        loss = tr.ctc_loss(logits, targets, il, tl).double().cpu()
        # check_ctc's bound: n frames' normalisers and steps, and the loss's own rounding
        assert abs(loss - ref) <= logits.shape[1] * 100 * E + E * ref + 1e-6, (float(loss), float(ref))
