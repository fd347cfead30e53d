"""Selection with many beams where the winners lie deep in few lists, evenly over all, or
tie: whatever bound the merge works from, the best of all candidates are chosen."""
import numpy as np
import pytest

import logits_oracle as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("v", [33, 256, 900, 2000, 6001])
@pytest.mark.parametrize("beams", [9, 15, 16, 17, 31, 32])
@pytest.mark.parametrize("owners", [1, 2, 3, 5, 9])
def test_deep_lists(rnet, cuda, v, beams, owners):
    """`owners` beams share the winners: each has beams / owners of them."""
    torch, batch = cuda, 3
    m = batch * beams
    r = np.random.default_rng(v * beams + owners)
    # all logits of a row distinct and on a grid, so that totals are apart or equal
    z = np.stack([r.permutation(v) for _ in range(m)]).astype(np.float32) / 64
    scores = np.full(m, -40.0, np.float32)
    for g in range(batch):
        scores[g * beams + r.permutation(beams)[:owners]] = -1.0
    fin = (r.random(m) < 0.1).astype(np.int32)
    for finished in (None, fin):
        zz, s = torch.from_numpy(z).cuda(), torch.from_numpy(scores).cuda()
        f = None if finished is None else torch.from_numpy(finished).cuda()
        out = torch.full((m,), 3.0, device="cuda")
        tok, par, done = (torch.full((m,), 55, dtype=torch.int32, device="cuda")
                          for _ in range(3))
        eos = -1 if f is None else 1
        rnet.call("rnet_beam_select", zz.data_ptr(), 0, v, s.data_ptr(),
                  None if f is None else f.data_ptr(), eos, out.data_ptr(), tok.data_ptr(),
                  par.data_ptr(), done.data_ptr(), batch, beams, v, None)
        torch.cuda.synchronize()
        # every row holds the same values: the normalisers are of the same numbers, added in
        # another order, and within their rounding; compare ranks by the exact common one
        lse = ref.logsumexp(z[0].astype(np.float64))
        for g in range(batch):
            rows = slice(g * beams, (g + 1) * beams)
            t = (scores[rows, None].astype(np.float64) + z[rows]) - lse
            if finished is not None:
                t[finished[rows] != 0] = -np.inf
                t[finished[rows] != 0, eos] = scores[rows][finished[rows] != 0]
            best = np.sort(t.reshape(-1))[::-1][:beams]
            p, k = par[rows].cpu().numpy(), tok[rows].cpu().numpy()
            got = t[p, k]
            # which of two totals that are equal but for rounding comes first is not held
            assert np.all(np.abs(got - best) <= 1e-6), (g, got, best)
            assert len({(a, b) for a, b in zip(p, k)}) == beams


@pytest.mark.parametrize("v", [40, 700, 2000, 6001])
@pytest.mark.parametrize("beams", [12, 17, 32])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_every_candidate_ties(rnet, cuda, v, beams, dtype):
    """Equal logits everywhere: more candidates than are ranked by counting. Some beams have
    ended, some have no score, some rows allow fewer tokens than there are beams."""
    torch, batch = cuda, 4
    m = batch * beams
    z = np.zeros((m, v), np.float32)
    scores, fin = np.full(m, -2.0, np.float32), np.zeros(m, np.int32)
    fin[beams + 1::5] = 1
    scores[2 * beams:3 * beams:2] = -np.inf
    z[3 * beams::3, 5:] = -np.inf
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    zz, s, f = (torch.from_numpy(a).cuda() for a in (z, scores, fin))
    zz = zz.to(t)
    out = torch.full((m,), 3.0, device="cuda")
    tok, par, done = (torch.full((m,), 55, dtype=torch.int32, device="cuda") for _ in range(3))
    rnet.call("rnet_beam_select", zz.data_ptr(), int(dtype == "bf16"), v, s.data_ptr(),
              f.data_ptr(), 3, out.data_ptr(), tok.data_ptr(), par.data_ptr(), done.data_ptr(),
              batch, beams, v, None)
    torch.cuda.synchronize()
    want = ref.select(z, scores, beams, 3, fin)
    assert want[4] > 1e-3
    np.testing.assert_array_equal(tok.cpu().numpy(), want[1])
    np.testing.assert_array_equal(par.cpu().numpy(), want[2])
    np.testing.assert_array_equal(done.cpu().numpy(), want[3])
