"""A decoder's captured step after the model's arithmetic has changed: what the graph
replays is what the launches one by one give."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

D, L, F, S, V, T = 64, 2, 128, 160, 256, 20
BATCH, BEAMS, STEPS = 2, 4, 6


@pytest.fixture
def model(rnet, rdata, cuda):
    cfg = rnet.ModelConfig.make(d_model=D, n_layers=L, d_ff=F, n_slots=S, top_k=2, vocab=V,
                                seq_len=T + STEPS + 4)
    p = rdata.init_params_normal(cfg, seed=6, std=0.05)
    rdata.split(cfg, p)["output"][:] *= 12.0
    m = rnet.Model(cfg, device=0, reference_init=False)
    m.set_params(p)
    dec = rnet.Decoder(m, BATCH * BEAMS)
    prompts = np.random.default_rng(6).integers(0, V, size=(BATCH, T)).astype(np.int32)
    yield m, dec, prompts
    dec.close()
    m.close()


def test_beam_search(cuda, model):
    torch = cuda
    m, dec, prompts = model
    tok = torch.from_numpy(prompts.reshape(-1)).cuda()

    def search(graph):
        seq = torch.zeros(dec.M, STEPS, dtype=torch.int32, device="cuda")
        ln, sc = torch.zeros(dec.M, dtype=torch.int32, device="cuda"), torch.zeros(dec.M).cuda()
        dec.prefill_beams(tok, T, BEAMS)
        dec.beam_search(BEAMS, STEPS, seq, ln, sc, use_graph=graph)
        m.synchronize()
        return seq.cpu().numpy(), sc.cpu().numpy()

    scores = []
    for precision in (0, 1, 0):
        m.set_precision(precision)
        graph, one_by_one = search(True), search(False)
        for a, b in zip(graph, one_by_one):
            np.testing.assert_array_equal(a, b)
        scores.append(graph[1])
    np.testing.assert_array_equal(scores[0], scores[2])
    assert np.any(scores[0] != scores[1])


def test_generate(cuda, model):
    torch = cuda
    m, dec, prompts = model
    tok = torch.from_numpy(np.repeat(prompts, BEAMS, 0).reshape(-1)).cuda()

    def last_logits(graph):
        dec.prefill(tok, T)
        if graph:
            dec.generate(STEPS, None)
        else:
            for _ in range(STEPS):
                dec.step(None)
        m.synchronize()
        return dec.outputs_host()[0].copy()

    for precision in (0, 1, 0):
        m.set_precision(precision)
        np.testing.assert_array_equal(last_logits(True), last_logits(False))
