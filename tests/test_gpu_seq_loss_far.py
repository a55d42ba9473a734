"""GPU tests of cfops_preference_loss where a reward is infinite: a term whose
weight is 0 is no part of the loss."""
import numpy as np
import pytest

from tests.test_gpu_seq_loss import EPS, run_preference, seqs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths", [[3, 4, 5, 6], [3000, 2000, 40, 50], [30] * 200], ids=lambda x: f"{len(x)}x{max(x)}")
def test_a_rejected_sequence_of_no_probability(lengths):
    """Its pair's loss is -log sigmoid(inf) = 0 and its gradients are 0; with label
    smoothing the loss is infinite."""
    off, tg, logp, ref, _ = seqs(lengths, 3, masked=0.0)
    logp[off[1]] = -np.inf
    loss, accuracy, margin, rewards, d = run_preference(off, tg, logp, ref, beta=0.3)
    x = logp.astype(np.float64) - ref.astype(np.float64)
    rew = np.array([0.3 * x[off[i]:off[i + 1]].sum() for i in range(len(lengths))])
    z = rew[::2] - rew[1::2]
    want = np.logaddexp(0, -z).mean()  # (of the first pair: 0)
    assert z[0] == np.inf and abs(loss - want) <= EPS * want + 2.0 ** -40
    assert rewards[1] == -np.inf and margin == np.inf
    assert not d[off[0]:off[2]].any() and np.isfinite(d).all() and d[off[2]:off[4]].all()
    assert run_preference(off, tg, logp, ref, beta=0.3, label_smoothing=0.1)[0] == np.inf


@pytest.mark.parametrize("form,want", [("hinge", np.inf), ("squared", np.inf), ("sigmoid", np.inf)])
def test_a_chosen_sequence_of_no_probability(form, want):
    off, tg, logp, ref, _ = seqs([3, 4, 5, 6], 3, masked=0.0)
    logp[off[0]] = -np.inf
    assert run_preference(off, tg, logp, ref, beta=0.3, form=form)[0] == want
