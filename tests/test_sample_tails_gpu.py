"""Sampling on the GPU from rows whose weights are a few units of the whole numbers that they are rounded to."""

import math
import os
import sys
from fractions import Fraction

import numpy as np
import pytest

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

from test_sample_gpu import BF, FF, clean, plain  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def shift_of(vocab):
    """Weights are round(w 2^shift), so that a row's sum stays under 2^63."""
    bits = (vocab - 1).bit_length()
    return 45 if bits <= 17 else 62 - bits


def whole_numbers(z, temperature, top_p, u):
    """The token, by whole-number weights of the row z (float64), exactly, and the logarithm of its share."""
    shift = shift_of(len(z))
    w = np.floor(np.exp((z - z.max()) / temperature) * 2.0 ** shift + 0.5).astype(np.int64)
    order = np.argsort(-z, kind="stable")
    mass = np.cumsum(w[order])
    target = max(1, math.ceil(Fraction(top_p) * int(mass[-1])))
    kept = order[:int(np.searchsorted(mass, target)) + 1]
    w[np.setdiff1d(order, kept, assume_unique=True)] = 0
    mass = np.cumsum(w)
    i = int(np.searchsorted(mass, math.floor(Fraction(u) * int(mass[-1])), side="right"))
    return i, float((z[i] - z.max()) / temperature) - math.log(int(mass[-1]) / 2 ** shift)


U = [0.0, 2.0 ** -30, 0.25, 0.5, 0.998, 1 - 2.0 ** -24]


@pytest.mark.parametrize("vocab,top_p", [(400, 1 - 2.0 ** -24), (3000, 1 - 2.0 ** -24), (50021, 0.9999999), (100000, 1 - 2.0 ** -24),
                                         (131072, 0.9999995), (262144, 0.9999), (1000003, 0.9999), (1000003, 0.999)])
@pytest.mark.parametrize("dtype", [FF, BF])
@pytest.mark.parametrize("more", [1, 2, 50])
def test_one_peak_over_a_flat_tail(vocab, top_p, dtype, more):
    """One likely token and a tail of equal ones, whose sum passes what top_p leaves by little or by half: each weighs `more`
    units over the least that does so, and is a little over half a unit under a whole number of them, so that rounding adds
    to the tail."""
    from heatvit_b200 import decode
    p = float(np.float32(top_p))
    scale = 2.0 ** shift_of(vocab)
    units = math.floor((1 - p) * scale / (vocab - 1) / p) + more
    away = -math.log((units - 0.47) / scale)
    if dtype == FF:
        low, temperature = -float(np.float32(away)), 1.0
    else:  # coarse logits: the temperature has the fine steps
        low, temperature = -24.0, float(np.float32(24.0 / away))
    assert abs(math.exp(low / temperature) * scale - (units - 0.47)) < 0.4, "a weight that rounds up"
    for peak in (0, vocab // 2, vocab - 1):
        z = torch.full((len(U), vocab), low, device="cuda", dtype=dtype)
        z[:, peak] = 0
        u = torch.tensor(U, device="cuda")
        token, logprob = decode.sample_tokens(z, u, temperature=temperature, top_p=p, return_logprob=True)
        want = [whole_numbers(z[0].double().cpu().numpy(), temperature, p, float(v)) for v in u.tolist()]
        assert token.tolist() == [w[0] for w in want]
        assert np.allclose(logprob.cpu().numpy(), [w[1] for w in want], rtol=2.0 ** -23, atol=2.0 ** -24)
        if peak == 0:
            # Rounded or not, the tail weighs under (units + 1) (vocab - 1) 2^-shift, 0.00102 at most, and what is kept of
            # it less, so that a peak which comes first is drawn by every number up to 0.998.
            assert token[:5].tolist() == plain(z, u, temperature=temperature, top_p=p)[2][:5].tolist() == [0] * 5


def test_flat_tails_after_other_rows():
    """The same rows between others, whose search has left its cut in shared memory, and in a captured call."""
    from heatvit_b200 import decode
    vocab, p, low = 50021, float(np.float32(0.9999999)), -26.76261329650879
    g = torch.Generator(device="cuda").manual_seed(1)
    z = torch.randn(300, vocab, generator=g, device="cuda")
    z[::2] = low
    z[::2, 0] = 0
    u = torch.rand(300, generator=g, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = decode.sample_tokens(z, u, top_p=p, top_k=torch.arange(300, device="cuda", dtype=torch.int32) % 2 * 100)
    for _ in range(2):
        graph.replay()
        assert bool((out[::2] == 0).all())


@pytest.mark.parametrize("temperature,top,low", [
    (0.9895793795585632, 31.55251121520996, -1.3288322664450902e-09), (0.9181880950927734, 29.276216506958008, -2.5560853433859165e-09),
    (1.0416868925094604, 33.21394729614258, -2.039854729574131e-09), (0.9366442561149597, 29.864686965942383, 1.5098072791985828e-09)])
def test_a_weight_of_half_a_unit(temperature, top, low):
    """A logit that weighs half a unit to the last bit counts for one in every sum or in none: between two likely ones it has the
    draw that falls on it."""
    from heatvit_b200 import decode
    assert all(float(np.float32(v)) == v for v in (temperature, top, low))
    z = torch.full((3, 2048), -math.inf, device="cuda")
    z[:, 0], z[:, 130], z[:, 300] = top, low, top
    token, logprob = decode.sample_tokens(z, torch.tensor([0.4999, 0.5, 0.5001], device="cuda"), temperature=temperature, return_logprob=True)
    # 2^45, one and 2^45 units: half of them, rounded down, is 2^45
    assert token.tolist() == [0, 130, 300]
    assert np.allclose(logprob.tolist(), [-math.log(2), -47 * math.log(2), -math.log(2)], rtol=2.0 ** -23)
