"""Limits of the decoder's beam search: refused before anything is launched."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("steps", [-1, 0, 2 ** 30 + 1, 2 ** 31 - 1])
def test_steps(rnet, rdata, cuda, steps):
    torch = cuda
    cfg = rnet.ModelConfig.make(d_model=64, n_layers=1, d_ff=64, n_slots=16, top_k=2, vocab=64,
                                seq_len=16)
    m = rnet.Model(cfg, device=0, reference_init=False)
    m.set_params(rdata.init_params_normal(cfg, seed=1, std=0.05))
    dec = rnet.Decoder(m, 2)
    dec.prefill_beams(torch.zeros(4, dtype=torch.int32, device="cuda"), 4, 2)
    out = torch.full((2,), 7, dtype=torch.int32, device="cuda")
    m.synchronize()
    n0, free = rnet.kernel_launches(), torch.cuda.mem_get_info()[0]
    with pytest.raises(rnet.RnetError, match="n_steps must be 1..2"):
        dec.beam_search(2, steps, out, out, out)
    assert rnet.kernel_launches() == n0 and torch.cuda.mem_get_info()[0] == free
    assert torch.all(out == 7)
    m.close()
