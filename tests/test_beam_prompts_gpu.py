"""Short prompts for many beams: prefill_beams equals a prefill of every stream with its
prompt. And a generation of no steps does nothing."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

D, L, F, S, V = 64, 2, 128, 160, 256


@pytest.fixture
def model(rnet, rdata, cuda):
    cfg = rnet.ModelConfig.make(d_model=D, n_layers=L, d_ff=F, n_slots=S, top_k=2, vocab=V,
                                seq_len=64)
    m = rnet.Model(cfg, device=0, reference_init=False)
    m.set_params(rdata.init_params_normal(cfg, seed=3, std=0.05))
    yield m
    m.close()


@pytest.mark.parametrize("t", [1, 2, 13, 14, 15])
@pytest.mark.parametrize("batch,beams", [(1, 32), (3, 5)])
def test_prompts(rnet, cuda, model, t, batch, beams):
    torch = cuda
    r = np.random.default_rng(t)
    prompts = r.integers(0, V, size=(batch, t)).astype(np.int32)
    got = []
    for copies in (beams, 1):
        dec = rnet.Decoder(model, batch * beams)
        p = prompts if copies > 1 else np.repeat(prompts, beams, 0)
        tok = torch.from_numpy(np.ascontiguousarray(p).reshape(-1)).cuda()
        if copies > 1:
            dec.prefill_beams(tok, t, beams)
        else:
            dec.prefill(tok, t)
        seq = torch.zeros(dec.M, 4, dtype=torch.int32, device="cuda")
        ln, sc = torch.zeros(dec.M, dtype=torch.int32, device="cuda"), torch.zeros(dec.M).cuda()
        first = dec.outputs_host()[0].copy()
        dec.beam_search(beams, 4, seq, ln, sc)
        model.synchronize()
        got.append((first, seq.cpu().numpy(), sc.cpu().numpy()))
        dec.close()
    # the same prompt in another number of rows: the GEMMs may split their sums differently
    for a, b in zip(*got):
        if a.dtype == np.int32:
            np.testing.assert_array_equal(a, b)
        else:
            assert np.all(np.abs(a - b) <= 1e-4 * np.abs(b).max())


def test_no_steps(rnet, cuda, model):
    torch = cuda
    dec = rnet.Decoder(model, 4)
    dec.prefill(torch.zeros(4 * 3, dtype=torch.int32, device="cuda"), 3)
    out = torch.full((4,), 77, dtype=torch.int32, device="cuda")
    model.synchronize()
    lg = dec.outputs_host()[0].copy()
    n0 = rnet.kernel_launches()
    for graph in (True, False):
        dec.generate(0, out, graph)
    assert rnet.kernel_launches() == n0
    model.synchronize()
    assert torch.all(out == 77)
    np.testing.assert_array_equal(dec.outputs_host()[0], lg)
    dec.close()
