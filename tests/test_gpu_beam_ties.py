"""mk_beam_select where logits that differ have one score in 64 bits: of one beam the larger logit first, then the lower token."""
import numpy as np
import pytest

from kv4_cases import beams64
from test_gpu_beam import Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,k", [(5000, 128), (151936, 16), (151936, 64), (30, 30)])
def test_logits_nearer_than_a_step_of_the_score(mk, V, k):
    """Two tokens to a logit, neighbours 2^-60 apart; the score's step is 2^-50 and more."""
    rng = np.random.default_rng(V)
    z = (rng.permutation(V) // 2 * 2.0 ** -60).astype(np.float32)
    steps = np.unique(z.astype(np.float64) - np.log(V) - 2)
    assert len(steps) < V // 4
    print("beams, near ties", V, k, flush=True)
    c = Call(mk, z[None], np.full(1, -2.0, np.float32), None, 0, 1, k)
    c.run()
    s, q, t = c.read()
    assert np.array_equal(t[0], np.lexsort((np.arange(V), -z))[:k]) and (q == 0).all()


@pytest.mark.parametrize("beams,V,k", [(2, 9001, 64), (3, 1300000, 128), (64, 40000, 16)])
def test_one_logit_that_is_infinite(mk, beams, V, k):
    """It counts as the largest float, beside which all other scores are one number: by beam, then by logit."""
    rng = np.random.default_rng(V)
    z = (np.round(4 * rng.standard_normal(V)) / 4).astype(np.float32)
    z[V // 3] = np.inf
    z = np.tile(z, (beams, 1))
    s = np.full(beams, -1.0, np.float32)
    print("beams, one infinite", beams, V, k, flush=True)
    c = Call(mk, z, s, None, 0, beams, k)
    c.run()
    got, q, t = c.read()
    want = beams64(z, s, None, 0, beams, k)[0][0]
    order = [v for v in np.lexsort((np.arange(V), -z[0])) if v != V // 3]
    plain = [(b, V // 3) for b in range(beams)] + [(0, int(v)) for v in order[:k]]
    assert [(b, v) for _, b, v in want] == plain[:k]
    assert list(zip(q[0].tolist(), t[0].tolist())) == plain[:k]
    assert (got[0][:min(beams, k)] == -1.0).all() and (got[0][beams:] == -np.finfo(np.float32).max).all()
