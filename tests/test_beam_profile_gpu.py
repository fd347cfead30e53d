"""A profiled search or generation asked for a graph runs launch by launch: the profile can
be read, counts every GEMM, and the outputs are the same."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

D, L, F, S, V, T, BATCH, BEAMS, STEPS = 64, 2, 128, 160, 256, 12, 2, 3, 6


@pytest.fixture
def pair(rnet, rdata, cuda):
    cfg = rnet.ModelConfig.make(d_model=D, n_layers=L, d_ff=F, n_slots=S, top_k=2, vocab=V,
                                seq_len=64)
    m = rnet.Model(cfg, device=0, reference_init=False)
    m.set_params(rdata.init_params_normal(cfg, seed=3, std=0.05))
    dec = rnet.Decoder(m, BATCH * BEAMS)
    yield m, dec
    dec.close()
    m.close()


def test_profiled(cuda, pair):
    torch = cuda
    m, dec = pair
    prompts = np.random.default_rng(3).integers(0, V, size=(BATCH, T)).astype(np.int32)
    tok = torch.from_numpy(prompts.reshape(-1)).cuda()
    seq = torch.zeros(dec.M, STEPS, dtype=torch.int32, device="cuda")
    ln = torch.zeros(dec.M, dtype=torch.int32, device="cuda")
    sc = torch.zeros(dec.M, device="cuda")
    out = torch.zeros(STEPS, dec.M, dtype=torch.int32, device="cuda")

    def run(profile):
        dec.prefill_beams(tok, T, BEAMS)
        m.profile_enable(profile)
        if profile:
            m.profile_read()  # of what was before
        dec.beam_search(BEAMS, STEPS, seq, ln, sc, use_graph=True)
        m.synchronize()
        gemms = [m.profile_read()["gemm"]["launches"]] if profile else []
        got = [seq.cpu().numpy().copy(), sc.cpu().numpy().copy()]
        dec.step(None)
        if profile:
            m.profile_read()
        dec.generate(STEPS, out, True)
        m.synchronize()
        gemms += [m.profile_read()["gemm"]["launches"]] if profile else []
        m.profile_enable(False)
        return got + [out.cpu().numpy().copy()], gemms

    first, _ = run(True)
    plain, _ = run(False)
    again, gemms = run(True)
    for a, b, c in zip(first, plain, again):
        np.testing.assert_array_equal(a, b)
        np.testing.assert_array_equal(a, c)
    # per step: mix, gates, scores, gate and up, down of every layer, and the head
    per_step = 5 * L + 1
    assert gemms == [per_step * (STEPS - 1), per_step * STEPS]
