"""A decoder's handle is destroyed before its model's, whatever order Python ends the two
objects in. The library's functions are stood in for, so this needs no GPU."""
import gc

import pytest


class Library:
    """Hands out handles and keeps the order of what is destroyed."""

    def __init__(self):
        self.next, self.ended = 100, []

    def _create(self, out):
        self.next += 1
        out._obj.value = self.next
        return 0

    def rnet_model_create(self, cfg, device, init, out):
        return self._create(out)

    def rnet_decoder_create(self, model, n, out):
        return self._create(out)

    def rnet_model_destroy(self, h):
        self.ended.append(("model", h.value))
        return 0

    def rnet_decoder_destroy(self, h):
        self.ended.append(("decoder", h.value))
        return 0

    def __getattr__(self, name):
        return lambda *a: 0


@pytest.fixture
def fake(rnet, monkeypatch):
    f = Library()
    monkeypatch.setattr(rnet, "lib", lambda: f)
    return f


def _pair(rnet):
    m = rnet.Model(rnet.ModelConfig.make(d_model=8, n_layers=1, d_ff=16, n_slots=4, top_k=2,
                                         vocab=16, seq_len=8))
    return m, rnet.Decoder(m, 2)


def test_the_model_closes_its_decoders(rnet, fake):
    m, d = _pair(rnet)
    other = rnet.Decoder(m, 4)
    m.close()
    assert sorted(fake.ended[:2]) == [("decoder", 102), ("decoder", 103)]
    assert fake.ended[2:] == [("model", 101)]
    d.close()
    other.close()
    m.close()
    assert len(fake.ended) == 3 and not d.handle and not other.handle


def test_a_closed_decoder_is_not_closed_again(rnet, fake):
    m, d = _pair(rnet)
    d.close()
    m.close()
    assert fake.ended == [("decoder", 102), ("model", 101)]


@pytest.mark.parametrize("first", ["model", "decoder"])
def test_a_collected_cycle(rnet, fake, first):
    m, d = _pair(rnet)
    ends = (m, d) if first == "model" else (d, m)
    del m, d
    for x in ends:  # what the collector does with the objects of a cycle, in this order
        type(x).__del__(x)
    ends = None
    gc.collect()
    assert fake.ended == [("decoder", 102), ("model", 101)]
