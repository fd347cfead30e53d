"""What the operators on logits and beams refuse: an error code, a message, no
launch and nothing written. Needs no GPU."""
import ctypes

import numpy as np
import pytest

F = ctypes.c_float


@pytest.fixture()
def buf():
    b = np.zeros(4096, np.float32)
    return b, b.ctypes.data + (-b.ctypes.data) % 16


def _refused(rnet, name, args, text, code=-1):
    n0 = rnet.kernel_launches()
    rc = getattr(rnet.lib(), name)(*args)
    assert rc == code, (rc, text)
    assert text in rnet.lib().rnet_last_error().decode()
    assert rnet.kernel_launches() == n0


TOPK = dict(logits=1, dtype=0, ld=8, tau=1.0, top=1, idx=1, lse=0, rows=2, vocab=8, k=2)
DISTILL = dict(logits=1, dtype=0, ld=8, t_idx=1, t_val=1, t_lse=0, targets=0, weight=0, tau=1.0,
               soft=1.0, hard=0.0, scale=1.0, row_loss=1, loss=0, dlogits=0, ldd=0, rows=2, vocab=8,
               k=2)
SELECT = dict(logits=1, dtype=0, ld=8, s_in=1, f_in=0, eos=-1, s=1, tok=1, par=1, fin=0, batch=1,
              beams=2, vocab=8)
REORDER = dict(src=1, dst=1, row=16, pitch=16, outer=1, opitch=0, par=1, batch=1, beams=2)
BACK = dict(tok=1, par=1, s=1, eos=-1, alpha=0.0, seq=1, ln=1, rk=1, steps=2, batch=1, beams=2)
POINTERS = {"logits", "top", "idx", "lse", "t_idx", "t_val", "t_lse", "targets", "weight",
            "row_loss", "loss", "dlogits", "s_in", "f_in", "s", "tok", "par", "fin", "src", "dst",
            "seq", "ln", "rk"}
ENTRY = {"rnet_topk_logits_forward": TOPK, "rnet_distill_topk_forward": DISTILL,
         "rnet_beam_select": SELECT, "rnet_beam_reorder": REORDER, "rnet_beam_backtrack": BACK}


def _args(entry, base, change):
    a = {**ENTRY[entry], **change}
    # pointers: 0 = null, n = base + (n - 1) bytes
    v = [None if k in POINTERS and x == 0 else ctypes.c_void_p(base + x - 1) if k in POINTERS
         else x for k, x in a.items()]
    return v + [None]


@pytest.mark.parametrize("entry,change,text", [
    *[("rnet_topk_logits_forward", {p: 0}, "null pointer") for p in ("logits", "top", "idx")],
    ("rnet_topk_logits_forward", dict(dtype=2), "dtype"),
    ("rnet_topk_logits_forward", dict(rows=-1), "bad size"),
    ("rnet_topk_logits_forward", dict(vocab=0), "bad size"),
    ("rnet_topk_logits_forward", dict(ld=7), "row pitch"),
    ("rnet_topk_logits_forward", dict(vocab=2 ** 30 + 1, ld=2 ** 31), "2^30"),
    ("rnet_topk_logits_forward", dict(k=0), "top_k"),
    ("rnet_topk_logits_forward", dict(k=9), "top_k"),
    ("rnet_topk_logits_forward", dict(vocab=100, ld=100, k=65), "top_k"),
    ("rnet_topk_logits_forward", dict(tau=0.0), "temperature"),
    ("rnet_topk_logits_forward", dict(tau=float("nan")), "temperature"),
    ("rnet_topk_logits_forward", dict(tau=float("inf")), "temperature"),
    ("rnet_topk_logits_forward", dict(tau=1e-45), "temperature"),
    ("rnet_topk_logits_forward", dict(logits=3), "aligned"),
    ("rnet_topk_logits_forward", dict(dtype=1, logits=2), "aligned"),
    ("rnet_topk_logits_forward", dict(lse=3), "aligned"),
    *[("rnet_distill_topk_forward", {p: 0}, "null pointer")
      for p in ("logits", "t_idx", "t_val", "row_loss")],
    ("rnet_distill_topk_forward", dict(dtype=-1), "dtype"),
    ("rnet_distill_topk_forward", dict(rows=-3), "bad size"),
    ("rnet_distill_topk_forward", dict(ld=1), "row pitch"),
    ("rnet_distill_topk_forward", dict(dlogits=2049, ldd=7), "row pitch"),
    ("rnet_distill_topk_forward", dict(ld=2 ** 61), "too large"),
    ("rnet_distill_topk_forward", dict(dlogits=2049, ldd=2 ** 61), "too large"),
    ("rnet_distill_topk_forward", dict(k=65), "top_k"),
    ("rnet_distill_topk_forward", dict(tau=-1.0), "temperature"),
    ("rnet_distill_topk_forward", dict(soft=float("inf")), "finite"),
    ("rnet_distill_topk_forward", dict(scale=float("nan")), "finite"),
    ("rnet_distill_topk_forward", dict(hard=0.5), "targets"),
    ("rnet_distill_topk_forward", dict(weight=2), "aligned"),
    ("rnet_distill_topk_forward", dict(dlogits=5, ldd=8), "overlaps"),
    ("rnet_distill_topk_forward", dict(dlogits=1, ldd=9), "overlaps"),
    *[("rnet_beam_select", {p: 0}, "null pointer") for p in ("logits", "s_in", "s", "tok", "par")],
    ("rnet_beam_select", dict(dtype=3), "dtype"),
    ("rnet_beam_select", dict(batch=-1), "bad size"),
    ("rnet_beam_select", dict(beams=0), "beams"),
    ("rnet_beam_select", dict(beams=33), "beams"),
    ("rnet_beam_select", dict(ld=7), "row pitch"),
    ("rnet_beam_select", dict(vocab=2 ** 30 + 1, ld=2 ** 31), "2^30"),
    ("rnet_beam_select", dict(eos=8), "eos"),
    ("rnet_beam_select", dict(eos=-2), "eos"),
    ("rnet_beam_select", dict(f_in=1, fin=1), "eos"),
    ("rnet_beam_select", dict(f_in=1, eos=0), "finished"),
    ("rnet_beam_select", dict(batch=2 ** 31 - 1), "too large"),
    ("rnet_beam_select", dict(tok=2), "aligned"),
    *[("rnet_beam_reorder", {p: 0}, "null pointer") for p in ("src", "dst", "par")],
    ("rnet_beam_reorder", dict(batch=65536), "batch"),
    ("rnet_beam_reorder", dict(outer=65536), "outer"),
    ("rnet_beam_reorder", dict(beams=33), "beams"),
    ("rnet_beam_reorder", dict(row=18, pitch=20), "multiples of 4"),
    ("rnet_beam_reorder", dict(src=2, dst=2), "multiples of 4"),
    ("rnet_beam_reorder", dict(pitch=12), "row pitch"),
    ("rnet_beam_reorder", dict(outer=2, opitch=16), "outer pitch"),
    ("rnet_beam_reorder", dict(dst=17), "overlaps"),
    ("rnet_beam_reorder", dict(pitch=2 ** 63), "too large"),
    ("rnet_beam_reorder", dict(row=2 ** 39, pitch=2 ** 39), "too long"),
    *[("rnet_beam_backtrack", {p: 0}, "null pointer")
      for p in ("tok", "par", "s", "seq", "ln", "rk")],
    ("rnet_beam_backtrack", dict(steps=0), "bad size"),
    ("rnet_beam_backtrack", dict(batch=-1), "bad size"),
    ("rnet_beam_backtrack", dict(steps=2 ** 30 + 1), "bad size"),
    ("rnet_beam_backtrack", dict(beams=40), "beams"),
    ("rnet_beam_backtrack", dict(alpha=float("nan")), "finite"),
    ("rnet_beam_backtrack", dict(seq=3), "aligned"),
    ("rnet_beam_backtrack", dict(), "overlap"),
    ("rnet_beam_backtrack", dict(seq=1025, tok=1029, par=2049), "overlap"),
])
def test_refused(rnet, buf, entry, change, text):
    _refused(rnet, entry, _args(entry, buf[1], change), text)
    assert not buf[0].any()


def test_refused_vocabulary(rnet, buf):
    a = _args("rnet_distill_topk_forward", buf[1], dict(vocab=262145, ld=262145))
    _refused(rnet, "rnet_distill_topk_forward", a, "262144", code=-7)
