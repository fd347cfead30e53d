"""A beam search needs logits of the streams' last tokens: after a prefill, a step or a
generation, not on a new decoder and not right after another search."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

D, L, F, S, V, T = 64, 2, 128, 160, 256, 20
BATCH, BEAMS, STEPS = 2, 3, 4


def test_search_after_search(rnet, rdata, cuda):
    torch = cuda
    cfg = rnet.ModelConfig.make(d_model=D, n_layers=L, d_ff=F, n_slots=S, top_k=2, vocab=V,
                                seq_len=64)
    m = rnet.Model(cfg, device=0, reference_init=False)
    m.set_params(rdata.init_params_normal(cfg, seed=2, std=0.05))
    dec = rnet.Decoder(m, BATCH * BEAMS)
    prompts = np.random.default_rng(2).integers(0, V, size=(BATCH, T)).astype(np.int32)
    tok = torch.from_numpy(prompts.reshape(-1)).cuda()
    seq = torch.full((dec.M, STEPS), -9, dtype=torch.int32, device="cuda")
    ln = torch.full((dec.M,), -9, dtype=torch.int32, device="cuda")
    sc = torch.full((dec.M,), 9.0, device="cuda")

    def refused():
        for t in (seq, ln, sc):
            t.fill_(-9)
        torch.cuda.synchronize()
        n0 = rnet.kernel_launches()
        with pytest.raises(rnet.RnetError, match="prefill or step first"):
            dec.beam_search(BEAMS, STEPS, seq, ln, sc)
        assert rnet.kernel_launches() == n0
        m.synchronize()
        assert all(torch.all(t == -9) for t in (seq, ln, sc))

    def search(**kw):
        dec.beam_search(BEAMS, STEPS, seq, ln, sc, **kw)
        m.synchronize()
        return seq.cpu().numpy().copy(), sc.cpu().numpy().copy()

    refused()
    for graph in (True, False):
        dec.prefill_beams(tok, T, BEAMS)
        first = search(use_graph=graph)
        refused()
        # the best sequence's last token, and on: as from a prefill of all tokens
        dec.step(None)
        on = search(use_graph=graph)
        refused()
        dec.generate(1, None, use_graph=graph)
        search(use_graph=graph)
        refused()
        dec.generate(2, None, use_graph=True)
        search(use_graph=graph)
        refused()
        whole = np.concatenate([prompts, first[0][::BEAMS]], axis=1).astype(np.int32)
        dec.prefill_beams(torch.from_numpy(np.ascontiguousarray(whole).reshape(-1)).cuda(),
                          T + STEPS, BEAMS)
        again = search(use_graph=graph)
        # decode and prefill round differently: the parity tolerance of the decode path
        assert np.all(np.abs(on[1] - again[1]) <= 1e-4 * np.abs(again[1]))
    dec.close()
    m.close()
