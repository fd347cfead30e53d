"""Where a row is cut: its first and last elements outside the 16-byte grid, the edges of
chunks and of the shares of CTAs and slices. One element a row stands out by 20, so that a
sum without it is off by orders of magnitude, and the sums are held to the depth that the
kernels' additions have.

Bounds count roundings (U = 2^-24). A sum's terms are added by a thread one after another,
at most DEPTH - 16 of them or of partial sums (a chunk's 32 values and two roundings a
chunk of 4096 for the selection; a thread's share of at most 128 elements for the
distillation), then over 32 lanes, the warps and the CTAs. A term's argument a moves it by 3 |a| U,
the exponential is within 4 U."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DEPTH = 160


def _places(v, offset, es):
    """Elements next to every place where a row of v elements, `offset` elements off the
    16-byte grid, can be cut."""
    n = 16 // es
    head = -offset % n
    at = set(range(16)) | set(range(v - 16, v))
    for chunk in (1024, 2048, 4096, 8192, 16384):  # of elements
        for start in (0, head):
            at |= {start + k * chunk + d for k in range(1, v // chunk + 1) for d in (-1, 0)}
    for c in range(2, 17):  # shares of CTAs: whole pieces, slices: whole 16s
        per, cut = -(-(v // n) // c), -(-(-(-v // c)) // 16) * 16
        for k in range(1, c):
            at |= {head + k * per * n + d for d in (-1, 0)} | {k * cut + d for d in (-1, 0)}
    return sorted(i for i in at if 0 <= i < v)


def _rows(torch, v, offset, dtype, few, seed, most=220):
    """Rows with one of the places raised each: [n, v] logits at their pitch, and the places.
    few: at most 140 rows, otherwise at least 150."""
    t, es = (torch.float32, 4) if dtype == "f32" else (torch.bfloat16, 2)
    r = np.random.default_rng(seed)
    at = _places(v, offset, es)
    if len(at) > most:
        ends = [i for i in at if i < 16 or i >= v - 16]
        inner = [i for i in at if 16 <= i < v - 16]
        at = ends + [inner[j] for j in np.sort(r.permutation(len(inner))[:most - len(ends)])]
    if few:
        at = [at[j] for j in np.sort(r.permutation(len(at))[:140])]
    else:
        at = (at * -(-150 // len(at)))[:max(150, len(at))]
    n, pad = len(at), 16 // es  # a pitch that keeps every row at the same offset
    ld = -(-v // pad) * pad + pad
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.full((n * ld + 16,), 30.0, dtype=t, device="cuda")
    z = torch.as_strided(buf, (n, v), (ld, 1), offset)
    z.copy_(torch.randn(n, v, device="cuda", generator=g).to(t))
    place = torch.tensor(at, device="cuda")
    z[torch.arange(n, device="cuda"), place] += 20.0
    return z, place


def _sum_bound(torch, z, tau):
    """(largest, log sum exp in 64 bits relative to it, relative bound of the sum)."""
    d = (z.double() - z.double().amax(1, keepdim=True)) / tau
    e = d.exp()
    s = e.sum(1)
    return d, e, s, (DEPTH + 4 + (e * 3 * d.abs()).sum(1) / s) * U


CASES = [(255, 1), (257, 3), (1001, 2), (1025, 5), (2049, 1), (4099, 7), (8191, 3), (8193, 0),
         (9001, 6), (20001, 4), (30001, 1), (50001, 0), (50001, 5), (100003, 3)]


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v,offset", CASES)
def test_records(rnet, cuda, v, offset, dtype, few):
    torch, k, tau = cuda, 3, 2.0
    z, place = _rows(torch, v, offset, dtype, few, v + offset)
    n = z.shape[0]
    top = torch.full((n, k), 9.0, device="cuda")
    idx = torch.full((n, k), 9, dtype=torch.int32, device="cuda")
    lse = torch.full((n,), 9.0, device="cuda")
    rnet.call("rnet_topk_logits_forward", z.data_ptr(), int(dtype == "bf16"), z.stride(0), tau,
              top.data_ptr(), idx.data_ptr(), lse.data_ptr(), n, v, k, None)
    torch.cuda.synchronize()
    assert torch.equal(idx[:, 0].long(), place)
    assert torch.equal(top, z.float().topk(k, 1)[0])
    _, _, s, bound = _sum_bound(torch, z, tau)
    m = z.double().amax(1) / tau
    want = m + s.log()
    # the quotient and the sum are rounded, the logarithm is within 4 U
    bound = bound + (m.abs() * 2 + want.abs() + s.log().abs() * 4 + 1) * U
    assert torch.all((lse.double() - want).abs() <= bound), ((lse.double() - want).abs() / bound).max()


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v,offset", CASES)
def test_selection(rnet, cuda, v, offset, dtype, few):
    """Each place in a beam of its own sequence: one beam, cut into slices where rows are few."""
    torch = cuda
    z, place = _rows(torch, v, offset, dtype, few, v + offset)
    d, _, s, bound = _sum_bound(torch, z, 1.0)
    for part in ((slice(0, 7), slice(60, 68), slice(0, 140)) if few else (slice(0, None),)):
        zz, at = z[part], place[part]
        n = len(at)
        score = torch.full((n,), -3.0, device="cuda")
        out = torch.full((n,), 9.0, device="cuda")
        tok, par = (torch.full((n,), 9, dtype=torch.int32, device="cuda") for _ in range(2))
        rnet.call("rnet_beam_select", zz.data_ptr(), int(dtype == "bf16"), z.stride(0),
                  score.data_ptr(), None, -1, out.data_ptr(), tok.data_ptr(), par.data_ptr(), None,
                  n, 1, v, None)
        torch.cuda.synchronize()
        assert torch.equal(tok.long(), at) and torch.all(par == 0)
        want = -3.0 - s[part].log()
        assert torch.all((out.double() - want).abs() <= bound[part] + want.abs() * 2 * U)


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("mode", ["soft", "mixed"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v,offset", CASES)
def test_distillation(rnet, cuda, v, offset, dtype, mode, few):
    torch, k, tau = cuda, 5, 1.5
    soft, hard = (1.0, 0.0) if mode == "soft" else (0.7, 0.3)
    z, place = _rows(torch, v, offset, dtype, few, v + offset, most=180)
    n = z.shape[0]
    g = torch.Generator(device="cuda").manual_seed(v)
    rows = torch.arange(n, device="cuda")
    # entries and labels next to the raised element, and anywhere; distinct in a row
    idx = (place[:, None] + torch.tensor([1, v // 2, v - 1, v // 3, v // 5], device="cuda")) % v
    val = torch.randn(n, k, device="cuda", generator=g)
    y = (place + 2) % v
    I, Y = idx.to(torch.int32).contiguous(), y.to(torch.int32)
    row, loss = torch.full((n,), 9.0, device="cuda"), torch.zeros(1, device="cuda")
    out = torch.full((n, z.stride(0)), 9.0, dtype=z.dtype, device="cuda")
    grad = torch.as_strided(out, (n, v), (z.stride(0), 1), 0)
    rnet.call("rnet_distill_topk_forward", z.data_ptr(), int(dtype == "bf16"), z.stride(0),
              I.data_ptr(), val.data_ptr(), None, Y.data_ptr(), None, tau, soft, hard, 1.0,
              row.data_ptr(), loss.data_ptr(), grad.data_ptr(), z.stride(0), n, v, k, None)
    torch.cuda.synchronize()
    d, e, s, rel = _sum_bound(torch, z, tau)
    logq = d - s.log()[:, None]
    q, d = e.div_(s[:, None]), d.abs_()
    t = val.double() / tau
    logp = torch.log_softmax(t, 1)
    p = logp.exp()
    lq = logq.gather(1, idx)
    want = soft * tau * tau * (p * (logp - lq)).sum(1)
    own = 32 + 8 * t.abs().amax(1)  # roundings of a record's probability
    bl = soft * tau * tau * ((p * (logp.abs() + lq.abs())).sum(1) * 16 * U + rel + own * U)
    ge = (q * soft * tau).scatter_add_(1, idx, -p * soft * tau)
    bg = soft * tau * q * (rel[:, None] + (own[:, None] + 4 * d) * U)
    bg.scatter_add_(1, idx, soft * tau * p * own[:, None] * U)
    del logq, q, d, e
    if hard:
        d, e, s, rel = _sum_bound(torch, z, 1.0)
        ly = d.gather(1, y[:, None])[:, 0] - s.log()
        want = want - hard * ly
        bl = bl + hard * (ly.abs() * 8 * U + rel)
        q = e.div_(s[:, None])
        bg += hard * q * (rel[:, None] + 4 * d.abs() * U)
        bg[rows, y] += hard * 4 * U
        ge += hard * q
        ge[rows, y] -= hard
        del q, d, e
    bl = bl + want.abs() * 4 * U
    assert torch.all((row.double() - want).abs() <= bl), ((row.double() - want).abs() / bl).max()
    assert abs(float(loss) - float(want.sum())) <= float(bl.sum() + want.sum().abs() * U)
    half = 0.0 if dtype == "f32" else 2.0 ** -8
    bg += ge.abs() * (4 * U + half) + 1e-37
    bad = (grad.double() - ge).abs() > bg
    assert not bad.any(), (bad.nonzero()[:4], ((grad.double() - ge).abs() / bg).max())
    assert torch.all(torch.as_strided(out, (n, z.stride(0) - v), (z.stride(0), 1), v) == 9.0)
