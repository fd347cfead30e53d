"""Rows whose logits tie and hold NaN or +inf at once: the selection's first pass takes
them as they are, so ties fill its queue while NaN lies among them. Records and beam
selection against the plain forms of logits_oracle.py, compared exactly."""
import numpy as np
import pytest

import logits_oracle as ref

pytestmark = pytest.mark.gpu

LOWEST = -3.3895313892515355e38  # of bf16, exact in fp32


def _tied(kind, n, v, share, seed):
    r = np.random.default_rng(seed)
    z = np.full((n, v), -1.25, np.float32)
    if kind == "masked":  # all but a few hold the lowest value of the type
        z[:] = LOWEST
        for i in range(n):
            z[i, r.permutation(v)[:5]] = r.integers(-64, 64, size=5) / 8.0
    elif kind == "steps":
        z[:] = np.round(r.normal(size=(n, v)) * 2)
    elif kind == "zeros":
        z[:] = 0.0
        z[:, ::3] = -0.0
    z[r.random((n, v)) < share] = np.nan
    z[n - 1, v // 2] = np.inf
    return z


def _up(torch, z, dtype, offset):
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    n, v = z.shape
    buf = torch.zeros(n * v + 8, dtype=t, device="cuda")
    view = buf[offset:offset + n * v].view(n, v)
    view.copy_(torch.from_numpy(z).cuda().to(t))
    return view


CASES = [(kind, share) for kind in ("constant", "masked", "steps", "zeros")
         for share in (0.1, 0.3, 0.6)]


# 512 threads a row, then 128
@pytest.mark.parametrize("rows", [4, 150])
@pytest.mark.parametrize("v", [5000, 40000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,share", CASES)
def test_records(rnet, cuda, kind, share, dtype, v, rows):
    torch = cuda
    z = np.tile(_tied(kind, 3, v, share, v), (-(-rows // 3), 1))[:rows]
    zz = _up(torch, z, dtype, v % 3)
    rnet.device_error(clear=True)
    for k in (3, 48, 64):
        top = torch.full((rows, k), 5.0, device="cuda")
        idx = torch.full((rows, k), 77, dtype=torch.int32, device="cuda")
        rnet.call("rnet_topk_logits_forward", zz.data_ptr(), int(dtype == "bf16"), v, 1.0,
                  top.data_ptr(), idx.data_ptr(), None, rows, v, k, None)
        assert rnet.device_error(clear=True) == 0
        t0, i0, _ = ref.topk(z[:3], k, 1.0)
        same = np.arange(rows) % 3
        np.testing.assert_array_equal(idx.cpu().numpy(), i0[same])
        np.testing.assert_array_equal(top.cpu().numpy().astype(np.float64), t0[same])


@pytest.mark.parametrize("batch,beams", [(1, 4), (2, 32), (9, 17)])
@pytest.mark.parametrize("v", [5000, 40000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,share", CASES)
def test_selection(rnet, cuda, kind, share, dtype, v, batch, beams):
    torch, m = cuda, batch * beams
    z = _tied(kind, m, v, share, v + beams)
    scores = (-np.arange(m) / 64.0).astype(np.float32)
    zz, s = _up(torch, z, dtype, 1), torch.from_numpy(scores).cuda()
    out = torch.full((m,), 3.0, device="cuda")
    tok, par = (torch.full((m,), 55, dtype=torch.int32, device="cuda") for _ in range(2))
    rnet.device_error(clear=True)
    rnet.call("rnet_beam_select", zz.data_ptr(), int(dtype == "bf16"), v, s.data_ptr(), None, -1,
              out.data_ptr(), tok.data_ptr(), par.data_ptr(), None, batch, beams, v, None)
    assert rnet.device_error(clear=True) == 0
    want = ref.select(z, scores, beams)
    # totals that differ lie further apart than the log-normalisers (of about 10) may be off
    assert want[4] > 1e-5
    np.testing.assert_array_equal(tok.cpu().numpy(), want[1])
    np.testing.assert_array_equal(par.cpu().numpy(), want[2])
