"""Backtracking's ranks where the power of the length leaves 64 bits, or the score is
0, infinite or NaN: every output row is written once, in a total order."""
import numpy as np
import pytest

import logits_oracle as ref

pytestmark = pytest.mark.gpu


def _want(tok, par, scores, beams, eos, alpha):
    """Order, lengths and ranks; the sequences from the plain form without a length power."""
    t, m = tok.shape
    rows = []
    for g in range(m // beams):
        one = []
        at = slice(g * beams, (g + 1) * beams)
        for j in range(beams):
            # one beam at a time, by ranking it alone
            only = np.full(beams, -np.inf, np.float32)
            only[j] = 1.0
            s, n, _ = ref.backtrack(tok[:, at], par[:, at], only, beams, eos, 0.0)
            x = float(ref.canon(scores[g * beams + j]))
            with np.errstate(over="ignore", divide="ignore"):
                r = x if x in (0.0, -np.inf) else x / np.power(float(n[0]), float(np.float32(alpha)))
            one.append((r, s[0], n[0]))
        order = sorted(range(beams), key=lambda j: (-one[j][0], j))
        rows += [one[j] for j in order]
    return [np.array(c) for c in zip(*rows)]


@pytest.mark.parametrize("t", [1, 9, 5000])
@pytest.mark.parametrize("alpha", [200.0, -200.0, 3e38, -3e38, 0.6])
@pytest.mark.parametrize("beams", [4, 8])
def test_ranks(rnet, cuda, t, alpha, beams):
    torch, m = cuda, 2 * beams
    r = np.random.default_rng(t + beams)
    tok = r.integers(1, 50, size=(t, m)).astype(np.int32)
    tok[r.random((t, m)) < 0.5 / t] = 0
    par = np.tile(np.arange(beams), (t, 2)).astype(np.int32)
    scores = (-3 * r.random(m)).astype(np.float32)
    scores[0], scores[1], scores[3] = -np.inf, 0.0, np.nan
    scores[beams + 1], scores[beams + 2], scores[beams + 3] = np.inf, -0.0, -np.inf
    want = _want(tok, par, scores, beams, 0, alpha)
    up = lambda a: torch.from_numpy(a).cuda()
    T, P, S = up(tok), up(par), up(scores)
    seq = torch.full((m, t), 99, dtype=torch.int32, device="cuda")
    ln = torch.full((m,), 99, dtype=torch.int32, device="cuda")
    rk = torch.full((m,), 99.0, device="cuda")
    rnet.call("rnet_beam_backtrack", T.data_ptr(), P.data_ptr(), S.data_ptr(), 0, alpha,
              seq.data_ptr(), ln.data_ptr(), rk.data_ptr(), t, 2, beams, None)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(seq.cpu().numpy(), want[1])
    np.testing.assert_array_equal(ln.cpu().numpy(), want[2])
    with np.errstate(over="ignore"):
        r0 = want[0].astype(np.float32)
    got = rk.cpu().numpy()
    far = ~np.isfinite(r0) | (r0 == 0)
    np.testing.assert_array_equal(got[far], r0[far])
    assert np.all(np.abs(got[~far] - want[0][~far]) <= 2 * ref.U * np.abs(want[0][~far]) + 1e-45)
