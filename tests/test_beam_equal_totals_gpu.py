"""Unequal logits whose totals are the same 64-bit number: scores so large that the logits
do not show, and logits so small that the log-normaliser hides them. The order is the
lower beam, the larger logit, the lower token, however a row is cut."""
import numpy as np
import pytest

import logits_oracle as ref

pytestmark = pytest.mark.gpu


def _want(z, scores, beams):
    z, s = ref.canon(z), ref.canon(scores)
    tokens, parents = [], []
    with np.errstate(invalid="ignore"):
        total = (s[:, None] + z) - ref.logsumexp(z)[:, None]
    for g in range(len(s) // beams):
        c = []
        for b in range(beams):
            i = g * beams + b
            best = np.argsort(-z[i], kind="stable")[:beams]
            c += [(-total[i, v], b, -z[i, v], v) for v in best if total[i, v] > -np.inf]
        c = sorted(c)[:beams]
        assert len(c) == beams
        parents += [b for _, b, _, _ in c]
        tokens += [v for _, _, _, v in c]
    return tokens, parents


# 1 x 4 x 20000 and 2 x 2 x 50001 are cut into slices
@pytest.mark.parametrize("batch,beams,v", [(1, 4, 20000), (2, 2, 50001), (1, 1, 40000),
                                           (40, 4, 5000), (3, 8, 300), (2, 32, 1500)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["large", "low", "denormal"])
def test_equal_totals(rnet, cuda, batch, beams, v, dtype, kind):
    torch, m = cuda, batch * beams
    r = np.random.default_rng(v + beams)
    z = np.round(r.normal(size=(m, v)) * 8).astype(np.float32) / 4  # on a grid: ties too
    scores = (-1.0 - np.arange(m)).astype(np.float32)
    if kind == "large":
        scores[::beams] = np.inf  # one beam, above all
    elif kind == "low":
        scores[:] = np.finfo(np.float32).min
    else:
        z *= 2.0 ** -120
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    zz = torch.from_numpy(z).cuda().to(t).contiguous()
    s = torch.from_numpy(scores).cuda()
    out = torch.full((m,), 3.0, device="cuda")
    tok, par = (torch.full((m,), 55, dtype=torch.int32, device="cuda") for _ in range(2))
    rnet.call("rnet_beam_select", zz.data_ptr(), int(dtype == "bf16"), v, s.data_ptr(), None, -1,
              out.data_ptr(), tok.data_ptr(), par.data_ptr(), None, batch, beams, v, None)
    torch.cuda.synchronize()
    tokens, parents = _want(zz.float().cpu().numpy(), scores, beams)
    np.testing.assert_array_equal(par.cpu().numpy(), parents)
    np.testing.assert_array_equal(tok.cpu().numpy(), tokens)
