"""Top-logit records and the distillation loss on the GPU, against the plain
64-bit forms and bounds of logits_oracle.py."""
import ctypes

import numpy as np
import pytest

import logits_oracle as ref

pytestmark = pytest.mark.gpu

TYPES = ["f32", "bf16"]


def _rows(torch, n, v, dtype, pad=0, offset=0, seed=0, spread=3.0):
    """Logits [n, v] inside a larger buffer: pitch v + pad, `offset` elements in."""
    r = np.random.default_rng(seed)
    z = (r.normal(size=(n, v)) * spread).astype(np.float32)
    return _place(torch, z, dtype, pad, offset)


def _place(torch, z, dtype, pad=0, offset=0, fill=7.0):
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    n, v = z.shape
    buf = torch.full((n * (v + pad) + offset + 8,), fill, dtype=t, device="cuda")
    view = buf[offset:offset + n * (v + pad)].view(n, v + pad)[:, :v]
    view.copy_(torch.from_numpy(z).cuda().to(t))
    return buf, view


def _np(t):
    return t.detach().float().cpu().numpy()


def _code(rnet, dtype):
    return rnet.DTYPE_F32 if dtype == "f32" else rnet.DTYPE_BF16


def _topk(rnet, torch, z, dtype, k, tau=1.0, with_lse=True, stream=None):
    n, v = z.shape
    top = torch.full((n, k), 5.0, device="cuda")
    idx = torch.full((n, k), 77, dtype=torch.int32, device="cuda")
    lse = torch.full((n,), 9.0, device="cuda")
    rnet.call("rnet_topk_logits_forward", z.data_ptr(), _code(rnet, dtype), z.stride(0), tau,
              top.data_ptr(), idx.data_ptr(), lse.data_ptr() if with_lse else None, n, v, k, stream)
    torch.cuda.synchronize()
    return top.cpu().numpy(), idx.cpu().numpy(), lse.cpu().numpy()


def _check_topk(rnet, torch, z, dtype, k, tau=1.0):
    top, idx, lse = _topk(rnet, torch, z, dtype, k, tau)
    t0, i0, l0 = ref.topk(_np(z), k, tau)
    np.testing.assert_array_equal(idx, i0)
    np.testing.assert_array_equal(top.astype(np.float64), t0)
    fin = np.isfinite(l0)
    np.testing.assert_array_equal(np.isfinite(lse), fin)
    bound = ref.lse_bound(l0, z.shape[1])
    assert np.all(np.abs(lse[fin] - l0[fin]) <= bound[fin]), np.max(np.abs(lse[fin] - l0[fin]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k,pad,offset", [
    (1, 1, 1, 0, 0), (3, 2, 2, 0, 0), (5, 7, 7, 2, 1), (64, 256, 16, 0, 0), (9, 256, 64, 0, 0),
    (9, 64, 64, 0, 0), (7, 255, 33, 1, 3), (33, 257, 5, 0, 0), (2, 1000, 40, 0, 1),
    (3, 1024, 64, 0, 0), (3, 1025, 64, 0, 0), (2, 4097, 31, 5, 1), (1, 20000, 64, 0, 0),
    (3, 50001, 20, 0, 0), (2, 100003, 64, 0, 1), (160, 9001, 10, 0, 0), (700, 2049, 8, 0, 0),
    (1, 262145, 7, 0, 0)])
def test_topk_records(rnet, cuda, dtype, n, v, k, pad, offset):
    _, z = _rows(cuda, n, v, dtype, pad, offset, seed=n + v + k)
    _check_topk(rnet, cuda, z, dtype, k, tau=1.0 if v % 2 else 2.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [256, 1024, 5000, 40000])
@pytest.mark.parametrize("kind", ["constant", "ascending", "descending", "steps", "one_lane",
                                  "masked", "specials", "zeros"])
def test_topk_hard_rows(rnet, cuda, dtype, v, kind):
    n, k = 4, 48
    r = np.random.default_rng(v)
    z = (r.normal(size=(n, v)) * 2).astype(np.float32)
    if kind == "constant":
        z[:] = -1.25
    elif kind == "ascending":
        z[:] = np.sort(z, axis=1)
    elif kind == "descending":
        z[:] = -np.sort(-z, axis=1)
    elif kind == "steps":  # many ties
        z[:] = np.round(z)
    elif kind == "one_lane":  # the largest ones all 32 (and 512) apart
        z[:, 5::32] += 40.0
        z[1, 3::512] += 80.0
    elif kind == "masked":  # fewer logits than places; a row without any
        keep = r.random((n, v)) < 20.0 / v
        z[~keep] = -np.inf
        z[2] = -np.inf
        z[3] = -np.inf
        z[3, v - 1] = np.float32(-3.0e38)
    elif kind == "specials":
        z[0, ::3] = np.nan
        z[1, 7] = np.inf
        z[1, 100] = np.inf
        z[2] = np.nan
        z[3, ::2] = -np.inf
    elif kind == "zeros":
        z[:] = 0.0
        z[:, ::2] = -0.0
        z[0] = -np.abs(z[0])
    _, zz = _place(cuda, z, dtype)
    _check_topk(rnet, cuda, zz, dtype, k)


def test_topk_rows_beyond_stay_and_lse_is_optional(rnet, cuda):
    torch = cuda
    _, z = _rows(torch, 6, 300, "f32", seed=1)
    top = torch.full((6, 4), 5.0, device="cuda")
    idx = torch.full((6, 4), 77, dtype=torch.int32, device="cuda")
    rnet.call("rnet_topk_logits_forward", z.data_ptr(), 0, 300, 1.0, top.data_ptr(),
              idx.data_ptr(), None, 4, 300, 4, None)
    torch.cuda.synchronize()
    assert torch.all(top[4:] == 5.0) and torch.all(idx[4:] == 77)
    np.testing.assert_array_equal(idx[:4].cpu().numpy(), ref.topk(_np(z)[:4], 4, 1.0)[1])


def test_topk_pitch_past_32_bits(rnet, cuda):
    """Two rows more than 2^32 elements apart."""
    torch = cuda
    v, ld = 300, (1 << 32) + 64
    buf = torch.empty(ld + v, dtype=torch.bfloat16, device="cuda")
    z = (np.random.default_rng(3).normal(size=(2, v))).astype(np.float32)
    rows = torch.as_strided(buf, (2, v), (ld, 1))
    rows.copy_(torch.from_numpy(z).cuda())
    _check_topk(rnet, torch, rows, "bf16", 12)


def _teacher(r, n, v, k, tau):
    """A record with padding, repeated indices and entries at -inf."""
    idx = r.integers(0, v, size=(n, k)).astype(np.int32)
    val = (r.normal(size=(n, k)) * 2).astype(np.float32)
    for i in range(n):
        if i % 4 == 1:
            idx[i, k // 2:] = -1
            val[i, k // 2:] = np.nan  # never looked at
        if i % 4 == 2 and k > 1:
            idx[i, 1] = idx[i, 0]
        if i % 4 == 3 and k > 2:
            val[i, 2] = -np.inf
    if n > 6:
        idx[6] = -1
    return idx, val


def _distill(rnet, torch, z, dtype, idx, val, tau, soft, hard, scale, t_lse=None, targets=None,
             weight=None, grad=True, in_place=False, pad=0, stream=None):
    n, v = z.shape
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    row_loss = torch.full((n,), 9.0, device="cuda")
    loss = torch.full((1,), 9.0, device="cuda")
    d = z if in_place else torch.full((n, v + pad), 7.0, dtype=t, device="cuda")
    up = lambda a, ty: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(ty).cuda()
    I, X, L = up(idx, torch.int32), up(val, torch.float32), up(t_lse, torch.float32)
    G, W = up(targets, torch.int32), up(weight, torch.float32)
    ptr = lambda a: None if a is None else a.data_ptr()
    rnet.call("rnet_distill_topk_forward", z.data_ptr(), _code(rnet, dtype), z.stride(0), ptr(I),
              ptr(X), ptr(L), ptr(G), ptr(W), tau, soft, hard, scale, row_loss.data_ptr(),
              loss.data_ptr(), d.data_ptr() if grad else None, d.stride(0) if grad else 0, n, v,
              idx.shape[1], stream)
    torch.cuda.synchronize()
    if pad and not in_place:
        assert torch.all(d[:, v:] == 7.0)
    return row_loss.cpu().numpy(), float(loss.item()), _np(d[:, :v])


def _check(dtype, got, want):
    row_loss, loss, d = got
    l0, g0, bl, bg = want
    fin = np.isfinite(l0)
    np.testing.assert_array_equal(row_loss[~fin], l0[~fin])
    assert np.all(np.abs(row_loss[fin] - l0[fin]) <= bl[fin]), \
        np.max((np.abs(row_loss - l0) - bl)[fin])
    if np.all(fin):
        assert abs(loss - l0.sum()) <= bl.sum() + abs(l0.sum()) * ref.U
    bound = bg + (np.abs(g0) * ref.BF16 if dtype == "bf16" else 0.0) + 1e-38
    bad = np.abs(d - g0) > bound
    assert not bad.any(), (np.argwhere(bad)[:4], np.max(np.abs(d - g0) - bound))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k,pad,offset", [
    (1, 1, 1, 0, 0), (4, 2, 2, 0, 1), (9, 7, 5, 3, 1), (70, 256, 16, 0, 0), (8, 255, 64, 1, 1),
    (5, 1000, 33, 0, 0), (8, 1024, 8, 0, 0), (7, 1025, 8, 0, 0), (3, 4099, 64, 2, 0),
    (5, 9000, 17, 0, 0), (2, 20001, 64, 0, 3), (3, 50001, 32, 0, 0), (2, 100003, 9, 1, 0),
    (1, 262144, 64, 0, 0), (300, 2000, 4, 0, 0)])
@pytest.mark.parametrize("mode", ["soft", "mixed"])
def test_distill(rnet, cuda, dtype, n, v, k, pad, offset, mode):
    r = np.random.default_rng(n + v + k)
    _, z = _rows(cuda, n, v, dtype, pad, offset, seed=n * v)
    idx, val = _teacher(r, n, v, k, 2.0)
    kw = {}
    tau, soft, hard = 2.0, 1.0, 0.0
    if mode == "mixed":
        kw["targets"] = r.integers(0, v, size=n).astype(np.int32)
        kw["targets"][::3] = -1
        kw["weight"] = np.where(np.arange(n) % 5 == 4, 0.0, r.random(n) + 0.5).astype(np.float32)
        tau, soft, hard = 1.5, 0.7, 0.3
    want = ref.distill(_np(z), idx, val, tau, soft, hard, 1.0 / n, **kw)
    got = _distill(rnet, cuda, z, dtype, idx, val, tau, soft, hard, 1.0 / n, pad=3, **kw)
    _check(dtype, got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [256, 1500, 30001])
def test_distill_with_the_teachers_normaliser(rnet, cuda, dtype, v):
    """Record and loss together: p = the teacher's own probabilities."""
    torch, n, k, tau = cuda, 12, 20, 2.0
    _, t = _rows(torch, n, v, dtype, seed=5)
    top, idx, lse = _topk(rnet, torch, t, dtype, k, tau)
    _, z = _rows(torch, n, v, dtype, seed=6)
    want = ref.distill(_np(z), idx, top, tau, 0.5, 0.0, 0.25, t_lse=lse)
    got = _distill(rnet, torch, z, dtype, idx, top, tau, 0.5, 0.0, 0.25, t_lse=lse)
    _check(dtype, got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v,pad", [(256, 0), (511, 3), (3001, 0), (40000, 8)])
def test_distill_in_place_and_loss_only(rnet, cuda, dtype, v, pad):
    torch, n, k = cuda, 20, 12
    r = np.random.default_rng(v)
    buf, z = _rows(torch, n, v, dtype, pad, 1, seed=v)
    idx, val = _teacher(r, n, v, k, 2.0)
    args = (dtype, idx, val, 2.0, 1.0, 0.0, 1.0)
    a = _distill(rnet, torch, z, *args)
    b = _distill(rnet, torch, z, *args, grad=False)
    np.testing.assert_array_equal(a[0], b[0])
    assert a[1] == b[1] and np.all(b[2] == 7.0)
    outside = buf.clone()
    torch.as_strided(outside, (n, v), (v + pad, 1), 1).fill_(0)
    c = _distill(rnet, torch, z, *args, in_place=True)
    np.testing.assert_array_equal(a[0], c[0])
    np.testing.assert_array_equal(a[2], c[2])
    after = buf.clone()
    torch.as_strided(after, (n, v), (v + pad, 1), 1).fill_(0)
    assert torch.equal(outside, after)  # nothing between or beyond the rows


@pytest.mark.parametrize("v", [200, 3000, 30000])
def test_distill_masked_rows_and_logits(rnet, cuda, v):
    torch, n, k = cuda, 8, 6
    r = np.random.default_rng(2)
    z = (r.normal(size=(n, v)) * 2).astype(np.float32)
    idx = np.stack([r.permutation(v - 2)[:k] for _ in range(n)]).astype(np.int32)
    val = r.normal(size=(n, k)).astype(np.float32)
    targets = r.integers(0, v - 2, size=n).astype(np.int32)
    weight = np.ones(n, np.float32)
    z[:, v - 1] = -np.inf          # a token that no row allows
    z[0], weight[0] = np.nan, 0.0  # padded rows may hold anything
    z[1], weight[1] = -np.inf, 0.0
    z[2] = -np.inf                 # no distribution
    z[3] = np.finfo(np.float32).min
    z[4, v // 2:] = np.finfo(np.float32).min
    idx[4, 0] = 1
    idx[5] = -1                    # an empty record and no label
    targets[5] = -1
    idx[6, 3] = v - 1              # the teacher wants what the student rules out
    _, zz = _place(torch, z, "f32")
    want = ref.distill(z, idx, val, 2.0, 0.6, 0.4, 1.0, targets=targets, weight=weight)
    got = _distill(rnet, torch, zz, "f32", idx, val, 2.0, 0.6, 0.4, 1.0, targets=targets,
                   weight=weight)
    assert np.isposinf(want[0][6])
    _check("f32", got, want)
    for row in (0, 1, 2, 5):
        assert got[0][row] == 0.0 and np.all(got[2][row] == 0.0)
    # an unmasked NaN or +inf is not hidden
    z[3, 5], z[7, 6] = np.nan, np.inf
    _, zz = _place(torch, z, "f32")
    got = _distill(rnet, torch, zz, "f32", idx, val, 2.0, 0.6, 0.4, 1.0, targets=targets,
                   weight=weight)
    assert np.isnan(got[0][3]) and np.isnan(got[0][7]) and np.all(np.isnan(got[2][3]))
    assert got[0][5] == 0.0 and np.all(got[2][5] == 0.0)  # its neighbours are as before


@pytest.mark.parametrize("v", [100, 900, 5000, 40000])
@pytest.mark.parametrize("tau", [0.01, 1.0, 100.0])
def test_distill_huge_logits_and_extreme_temperatures(rnet, cuda, v, tau):
    """Logits up to the largest numbers, whose products with 1 / temperature leave
    fp32: only their differences count."""
    torch, n, k = cuda, 6, 5
    r = np.random.default_rng(v)
    z = (r.normal(size=(n, v)) * 2).astype(np.float32)
    big = np.float32(3.0e38)
    z[0, 3], z[0, 7] = big, big
    z[1] = -big
    z[2, ::2] = -big
    z[3, 1:] = -np.inf
    z[3, 0] = big
    z[4] = np.float32(1e35)
    idx = np.tile(np.array([3, 7, 0, 9, 11], np.int32), (n, 1))
    idx[3] = [0, -1, -1, -1, -1]
    idx[0, 2:] = -1
    val = r.normal(size=(n, k)).astype(np.float32)
    targets = np.array([7, 1, 1, 0, 2, 3], np.int32)
    _, zz = _place(torch, z, "f32")
    want = ref.distill(z, idx, val, tau, 0.6, 0.4, 1.0, targets=targets)
    got = _distill(rnet, torch, zz, "f32", idx, val, tau, 0.6, 0.4, 1.0, targets=targets)
    _check("f32", got, want)


@pytest.mark.parametrize("v", [100, 900, 5000, 40000])
@pytest.mark.parametrize("tau", [1e-4, 0.3, 1.0, 1e4])
def test_distill_logits_of_every_magnitude(rnet, cuda, v, tau):
    """Rows at +-10^e: the rounding of the largest logit over the temperature, far
    above 1 from 10^8 on, shows in no term."""
    torch, k = cuda, 4
    r = np.random.default_rng(v + 1)
    sizes = [s * 10.0 ** e for e in (3, 5, 7, 8, 9, 10, 12, 17, 25, 29, 31) for s in (1, -1)]
    n = len(sizes)
    z = np.zeros((n, v), np.float32)
    for i, b in enumerate(sizes):
        # some masked further down, some in another part of the row near the largest
        z[i] = np.float32(b) + (r.normal(size=v) * 2).astype(np.float32)
        z[i, v // 3: v // 2] = -np.inf
        z[i, v // 2: v // 2 + 5] = np.float32(b) * np.float32(1 + 1e-6)
        z[i, -3:] = np.float32(-3e38)
    idx = np.tile(np.array([1, v // 2 + 1, 0, -1], np.int32), (n, 1))
    val = r.normal(size=(n, k)).astype(np.float32)
    targets = np.full(n, v // 2 + 2, np.int32)
    _, zz = _place(torch, z, "f32")
    for soft, hard in ((0.6, 0.4), (1.0, 0.0), (0.0, 1.0)):
        want = ref.distill(z, idx, val, tau, soft, hard, 1.0, targets=targets)
        got = _distill(rnet, torch, zz, "f32", idx, val, tau, soft, hard, 1.0, targets=targets)
        _check("f32", got, want)


def test_distill_reports_indices_beyond_the_vocabulary(rnet, cuda):
    torch, n, v, k = cuda, 5, 300, 4
    r = np.random.default_rng(1)
    _, z = _rows(torch, n, v, "f32", seed=1)
    idx, val = r.integers(0, v, size=(n, k)).astype(np.int32), np.zeros((n, k), np.float32)
    targets = np.zeros(n, np.int32)
    rnet.device_error(clear=True)
    want = ref.distill(_np(z), idx, val, 1.0, 1.0, 1.0, 1.0, targets=targets)
    _check("f32", _distill(rnet, torch, z, "f32", idx, val, 1.0, 1.0, 1.0, 1.0, targets=targets),
           want)
    assert rnet.device_error(clear=True) == 0
    idx[1, 2], targets[3] = v, 1 << 30
    want = ref.distill(_np(z), idx, val, 1.0, 1.0, 1.0, 1.0, targets=targets)
    _check("f32", _distill(rnet, torch, z, "f32", idx, val, 1.0, 1.0, 1.0, 1.0, targets=targets),
           want)
    assert rnet.device_error(clear=True) == 2


@pytest.mark.parametrize("v", [61, 1400])
def test_distill_gradient_against_differences(rnet, cuda, v):
    """Central differences of the 64-bit loss: (L(z+h) - L(z-h)) / 2h is within
    h^2 max|L'''| / 6 of the derivative; the third derivative of log sum exp in
    one logit is below 0.1 / tau^3, so with h = 1e-3 that is below 2e-8, and the
    64-bit rounding of L / 2h below 1e-11."""
    torch, n, k, tau, soft, hard = cuda, 3, 7, 1.25, 0.8, 0.5
    r = np.random.default_rng(v)
    _, zz = _rows(torch, n, v, "f32", seed=v)
    z = _np(zz).astype(np.float64)
    idx, val = _teacher(r, n, v, k, tau)
    targets = r.integers(0, v, size=n).astype(np.int32)
    kw = dict(targets=targets)
    _, _, d = _distill(rnet, torch, zz, "f32", idx, val, tau, soft, hard, 1.0, **kw)
    bound = ref.distill(z, idx, val, tau, soft, hard, 1.0, **kw)[3]
    h = 1e-3
    for row in range(n):
        for j in list(r.integers(0, v, size=6)) + [int(idx[row, 0]), int(targets[row])]:
            one = lambda s: ref.distill(z[row:row + 1] + s * h * (np.arange(v) == j), idx[row:row + 1],
                                        val[row:row + 1], tau, soft, hard, 1.0,
                                        targets=targets[row:row + 1])[0][0]
            fd = (one(1) - one(-1)) / (2 * h)
            assert abs(d[row, j] - fd) <= bound[row, j] + 3e-8, (row, j)


def test_two_streams_at_once_and_a_replayed_graph(rnet, cuda):
    """Calls on two streams do not share anything, and a captured call replays
    on new contents."""
    torch, n, v, k = cuda, 64, 30001, 16
    r = np.random.default_rng(0)
    idx, val = _teacher(r, n, v, k, 2.0)
    zs = [_rows(torch, n, v, "f32", seed=s)[1] for s in (1, 2)]
    I, X = torch.from_numpy(idx).cuda(), torch.from_numpy(val).cuda()
    alone = [_distill(rnet, torch, z, "f32", idx, val, 2.0, 1.0, 0.0, 1.0) for z in zs]
    recs = [_topk(rnet, torch, z, "f32", k) for z in zs]
    streams = [torch.cuda.Stream() for _ in zs]
    outs = []
    for z, s in zip(zs, streams):
        o = [torch.empty(n, device="cuda"), torch.empty(1, device="cuda"), torch.empty_like(z),
             torch.empty(n, k, device="cuda"),
             torch.empty(n, k, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda")]
        outs.append(o)
    torch.cuda.synchronize()

    def both(z, o, s):
        rnet.call("rnet_distill_topk_forward", z.data_ptr(), 0, z.stride(0), I.data_ptr(),
                  X.data_ptr(), None, None, None, 2.0, 1.0, 0.0, 1.0, o[0].data_ptr(),
                  o[1].data_ptr(), o[2].data_ptr(), o[2].stride(0), n, v, k, s.cuda_stream)
        rnet.call("rnet_topk_logits_forward", z.data_ptr(), 0, z.stride(0), 1.0, o[3].data_ptr(),
                  o[4].data_ptr(), o[5].data_ptr(), n, v, k, s.cuda_stream)

    def check(o, a, t):
        np.testing.assert_array_equal(o[0].cpu().numpy(), a[0])
        assert float(o[1]) == a[1]
        np.testing.assert_array_equal(_np(o[2]), a[2])
        np.testing.assert_array_equal(o[4].cpu().numpy(), t[1])
        np.testing.assert_array_equal(o[5].cpu().numpy(), t[2])

    for _ in range(3):
        for z, o, s in zip(zs, outs, streams):
            both(z, o, s)
    torch.cuda.synchronize()
    for o, a, t in zip(outs, alone, recs):
        check(o, a, t)
    # capture on one input, replay on the other's contents
    z = zs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=streams[0]):
        both(z, outs[0], streams[0])
    z.copy_(zs[1])
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    check(outs[0], alone[1], recs[1])


def test_empty_batches(rnet, cuda):
    torch = cuda
    x = torch.full((4,), 3.0, device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    rnet.call("rnet_topk_logits_forward", x.data_ptr(), 0, 4, 1.0, x.data_ptr(), i.data_ptr(),
              None, 0, 4, 2, None)
    loss = torch.full((1,), 9.0, device="cuda")
    rnet.call("rnet_distill_topk_forward", x.data_ptr(), 0, 4, i.data_ptr(), x.data_ptr(), None,
              None, None, 1.0, 1.0, 0.0, 1.0, x.data_ptr(), loss.data_ptr(), None, 0, 0, 4, 2, None)
    torch.cuda.synchronize()
    assert torch.all(x == 3.0) and float(loss) == 0.0
