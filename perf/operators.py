"""Measured cases of the operators that work on a model's logits and on the
beams chosen from them:

  topk       a teacher's record: the largest logits of each row, with the
             row's log-normaliser
  distill    the loss of a student against such a record and its gradient
  select     one step of beam search: the best continuations over all beams
             and the vocabulary
  reorder    the recurrent state of the decoder's streams, in place, in the
             order of the chosen parents
  backtrack  the token sequences behind the last beams, ranked

`own` switches between the library's calls and the plain form of the same
operator (elementary torch operations).
"""
import importlib
import math

import torch

own = False

INF = float("inf")
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODE = {"f32": 0, "bf16": 1}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a byte-level teacher run over one training batch (64 x 256 tokens)
        dict(name="topk_batch", op="topk", rows=16384, vocab=256, k=16, dtype="f32", tau=2.0),
        # a teacher with a large, odd vocabulary that answers in bf16
        dict(name="topk_wide_bf16", op="topk", rows=1024, vocab=100003, k=64, dtype="bf16",
             tau=1.0),
        # distillation on one short sequence: latency
        dict(name="distill_sequence", op="distill", rows=256, vocab=256, k=8, dtype="f32",
             tau=2.0, hard=0.0),
        # the training batch of the byte-level model, mixed with the labels' loss
        dict(name="distill_batch", op="distill", rows=16384, vocab=256, k=16, dtype="f32",
             tau=2.0, hard=0.3),
        # a large, odd vocabulary in bf16
        dict(name="distill_wide_bf16", op="distill", rows=4096, vocab=50001, k=32, dtype="bf16",
             tau=1.5, hard=0.0),
        # one prompt, four beams: latency
        dict(name="select_prompt", op="select", batch=1, beams=4, vocab=256, dtype="f32"),
        # 256 streams of the byte-level decoder
        dict(name="select_streams", op="select", batch=32, beams=8, vocab=256, dtype="f32"),
        # the same streams over a large, odd vocabulary
        dict(name="select_wide", op="select", batch=32, beams=8, vocab=50001, dtype="f32"),
        # state of one prompt's beams in a one-layer model of width 64
        dict(name="reorder_prompt", op="reorder", outer=1, batch=1, beams=4, row=15 * 64),
        # state of 256 streams in the 8-layer model of width 512
        dict(name="reorder_streams", op="reorder", outer=8, batch=32, beams=8, row=15 * 512),
        # sequences of 256 streams after 256 steps
        dict(name="backtrack_streams", op="backtrack", steps=256, batch=32, beams=8),
        # a long answer of a few prompts
        dict(name="backtrack_long", op="backtrack", steps=4096, batch=4, beams=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["topk", "distill", "select", "reorder", "backtrack"])
    if op == "topk":
        vocab = _log(rng, 2, 100003)
        return dict(op=op, rows=_log(rng, 1, min(16384, 1024 * 100003 // vocab)), vocab=vocab,
                    k=min(vocab, _log(rng, 1, 64)), dtype=rng.choice(["f32", "bf16"]),
                    tau=rng.choice([1.0, 2.0, 4.0]))
    if op == "distill":
        vocab = _log(rng, 2, 100003)
        return dict(op=op, rows=_log(rng, 1, min(16384, 2048 * 50001 // vocab)), vocab=vocab,
                    k=min(vocab, _log(rng, 1, 64)), dtype=rng.choice(["f32", "bf16"]),
                    tau=rng.choice([1.0, 2.0, 4.0]), hard=rng.choice([0.0, 0.3]))
    if op == "select":
        vocab = _log(rng, 2, 100003)
        beams = _log(rng, 1, 32)
        most = max(1, min(64, 256 * 50001 // (vocab * beams)))
        return dict(op=op, batch=_log(rng, 1, most), beams=beams, vocab=vocab,
                    dtype=rng.choice(["f32", "bf16"]))
    if op == "reorder":
        outer, beams, row = _log(rng, 1, 24), _log(rng, 2, 32), _log(rng, 16, 30720)
        most = max(1, min(64, 8 * 256 * 15 * 512 // (outer * beams * row)))
        if outer * beams * row > 8 * 256 * 15 * 512:
            outer = 1
        return dict(op=op, outer=outer, batch=_log(rng, 1, most), beams=beams, row=row)
    steps, beams = _log(rng, 1, 4096), _log(rng, 1, 32)
    return dict(op=op, steps=steps, batch=_log(rng, 1, max(1, min(64, 65536 // (steps * beams)))),
                beams=beams)


def work(case):
    c = case
    if c["op"] in ("topk", "distill"):
        n = c["rows"] * c["vocab"]
        es = 4 if c["dtype"] == "f32" else 2
        if c["op"] == "topk":
            return {"bytes": n * es + c["rows"] * (8 * c["k"] + 4), "flops": 3 * n}
        return {"bytes": 2 * n * es + c["rows"] * (8 * c["k"] + 12), "flops": 8 * n}
    m = c["batch"] * c["beams"]
    if c["op"] == "select":
        n = m * c["vocab"]
        return {"bytes": n * (4 if c["dtype"] == "f32" else 2) + 24 * m, "flops": 3 * n}
    if c["op"] == "reorder":
        # rows whose parent is another row are written; their distinct parents are read
        w = c["beams"]
        moved = 1.0 - 1.0 / w
        read = min(moved, 1.0 - (1.0 - 1.0 / w) ** w)
        return {"bytes": c["outer"] * m * c["row"] * 4.0 * (moved + read) + 4 * m, "flops": 0}
    return {"bytes": 12 * c["steps"] * m + 12 * m, "flops": 0}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)

    def rand(*s):
        return torch.rand(*s, device="cuda", generator=g)

    def normal(*s):
        return torch.randn(*s, device="cuda", generator=g)

    def ints(hi, *s):
        return torch.randint(0, hi, s, device="cuda", generator=g, dtype=torch.int32)

    s = {"case": c}
    if c["op"] in ("topk", "distill"):
        n, v, k, t = c["rows"], c["vocab"], c["k"], TYPES[c["dtype"]]
        z = normal(n, v) * 3.0
        if c["op"] == "topk":
            z[:, v // 3] = -INF  # a token that the teacher's masks rule out
            s["logits"] = z.to(t)
            s["top"] = torch.empty(n, k, device="cuda")
            s["idx"] = torch.empty(n, k, device="cuda", dtype=torch.int32)
            s["lse"] = torch.empty(n, device="cuda")
            return s
        s["logits"] = z.to(t)
        z += normal(n, v)  # a teacher near the student
        top, idx = z.topk(k, dim=1)
        del z
        idx = idx.to(torch.int32)
        short = rand(n, 1) < 0.1  # records with fewer entries than the others
        idx[short & (torch.arange(k, device="cuda")[None, :] >= max(1, k // 2))] = -1
        s["idx"], s["top"] = idx.contiguous(), top.float().contiguous()
        s["targets"] = ints(v, n)
        s["targets"][rand(n) < 0.05] = -1  # no label
        s["weight"] = (rand(n) >= 0.1).float()  # padded positions weigh nothing
        s["scale"] = 1.0 / n
        s["row_loss"] = torch.empty(n, device="cuda")
        s["loss"] = torch.empty(1, device="cuda")
        s["dlogits"] = torch.empty_like(s["logits"])
        return s
    b, w = c["batch"], c["beams"]
    if c["op"] == "select":
        z = normal(b * w, c["vocab"]) * 2.5
        z[:, c["vocab"] // 2] = -INF  # a banned token
        s["logits"] = z.to(TYPES[c["dtype"]])
        s["scores"] = (-6.0 - rand(b, w) * 4.0).sort(dim=1, descending=True)[0].reshape(-1).contiguous()
        s["finished"] = (rand(b * w) < 0.1).to(torch.int32)
        s["eos"] = 0
        s["out_scores"] = torch.empty(b * w, device="cuda")
        s["out"] = [torch.empty(b * w, device="cuda", dtype=torch.int32) for _ in range(3)]
        return s
    if c["op"] == "reorder":
        s["state"] = normal(c["outer"], b * w, c["row"])
        s["parents"] = ints(w, b * w)
        return s
    t = c["steps"]
    s["eos"] = 0
    s["tokens"] = ints(256, t, b * w) + 1
    s["tokens"][rand(t, b * w) < 0.5 / t] = 0
    s["parents"] = ints(w, t, b * w)
    s["scores"] = (-rand(b * w) * 2.0 * t - 1.0).contiguous()
    s["sequences"] = torch.empty(b * w, t, device="cuda", dtype=torch.int32)
    s["lengths"] = torch.empty(b * w, device="cuda", dtype=torch.int32)
    s["ranked"] = torch.empty(b * w, device="cuda")
    return s


ALPHA = 0.6  # length normalisation of the ranking


def run(state):
    c = state["case"]
    if own:
        return _OWN[c["op"]](state, c)
    return _PLAIN[c["op"]](state, c)


# ------------------------------------------------------------------ the library's calls
def _lib():
    return importlib.import_module("resonance-net_b200")


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_topk(s, c):
    _lib().call("rnet_topk_logits_forward", s["logits"].data_ptr(), CODE[c["dtype"]], c["vocab"],
                c["tau"], s["top"].data_ptr(), s["idx"].data_ptr(), s["lse"].data_ptr(), c["rows"],
                c["vocab"], c["k"], _stream())
    return {"top": s["top"], "idx": s["idx"], "lse": s["lse"]}


def _own_distill(s, c):
    _lib().call("rnet_distill_topk_forward", s["logits"].data_ptr(), CODE[c["dtype"]], c["vocab"],
                s["idx"].data_ptr(), s["top"].data_ptr(), None,
                s["targets"].data_ptr() if c["hard"] else None, s["weight"].data_ptr(), c["tau"],
                1.0 - c["hard"], c["hard"], s["scale"], s["row_loss"].data_ptr(),
                s["loss"].data_ptr(), s["dlogits"].data_ptr(), c["vocab"], c["rows"], c["vocab"],
                c["k"], _stream())
    return {"row_loss": s["row_loss"], "loss": s["loss"], "dlogits": s["dlogits"]}


def _own_select(s, c):
    tokens, parents, finished = s["out"]
    _lib().call("rnet_beam_select", s["logits"].data_ptr(), CODE[c["dtype"]], c["vocab"],
                s["scores"].data_ptr(), s["finished"].data_ptr(), s["eos"],
                s["out_scores"].data_ptr(), tokens.data_ptr(), parents.data_ptr(),
                finished.data_ptr(), c["batch"], c["beams"], c["vocab"], _stream())
    return {"scores": s["out_scores"], "tokens": tokens, "parents": parents, "finished": finished}


def _own_reorder(s, c):
    x, row = s["state"], 4 * c["row"]
    _lib().call("rnet_beam_reorder", x.data_ptr(), x.data_ptr(), row, row, c["outer"],
                row * c["batch"] * c["beams"], s["parents"].data_ptr(), c["batch"], c["beams"],
                _stream())
    return {"state": x}


def _own_backtrack(s, c):
    _lib().call("rnet_beam_backtrack", s["tokens"].data_ptr(), s["parents"].data_ptr(),
                s["scores"].data_ptr(), s["eos"], ALPHA, s["sequences"].data_ptr(),
                s["lengths"].data_ptr(), s["ranked"].data_ptr(), c["steps"], c["batch"],
                c["beams"], _stream())
    return {"sequences": s["sequences"], "lengths": s["lengths"], "ranked": s["ranked"]}


# ------------------------------------------------------------------ plain forms
def _finite(x):
    """fp32 values with NaN as -inf, +inf as the largest number, and one zero."""
    return torch.nan_to_num(x.float(), nan=-INF, posinf=torch.finfo(torch.float32).max,
                            neginf=-INF) + 0.0


def _top_rows(x, k):
    """The k largest of each row, ties to the lowest index: (values, indices)."""
    i = x.view(torch.int32)
    o = (i ^ ((i >> 31) & 0x7FFFFFFF)).to(torch.int64)
    at = 0xFFFFFFFF - torch.arange(x.shape[1], device=x.device)
    top = ((o << 32) | at).topk(k, dim=1)[0]
    idx = 0xFFFFFFFF - (top & 0xFFFFFFFF)
    return x.gather(1, idx), idx


def _plain_topk(s, c):
    x = _finite(s["logits"])
    top, idx = _top_rows(x, c["k"])
    idx = torch.where(top > -INF, idx, -1).to(torch.int32)
    m = x.amax(1, keepdim=True)
    m = torch.where(m > -INF, m, 0.0)
    lse = (m[:, 0] / c["tau"]) + ((x - m) / c["tau"]).exp().sum(1).log()
    return {"top": top, "idx": idx, "lse": lse}


def _plain_distill(s, c):
    z, tau, hard = s["logits"].float(), c["tau"], c["hard"]
    w = s["weight"]
    rows = torch.arange(z.shape[0], device=z.device)
    m = z.amax(1, keepdim=True)
    e = ((z - m) / tau).exp()
    total = e.sum(1, keepdim=True)
    # teacher: softmax over the entries of the record
    has = s["idx"] >= 0
    at = s["idx"].clamp(min=0).long()
    t = torch.where(has, s["top"] / tau, -INF)
    tm = t.amax(1, keepdim=True)
    te = (t - tm).exp()
    ts = te.sum(1, keepdim=True)
    p = te / ts
    logp = torch.where(has, t - tm - ts.log(), 0.0)
    logq = (z.gather(1, at) - m) / tau - total.log()
    loss = (1.0 - hard) * tau * tau * torch.where(has, p * (logp - logq), 0.0).sum(1)
    grad = e.div_(total).scatter_add_(1, at, -p).mul_((1.0 - hard) * tau)
    if hard:
        e1 = (z - m).exp()
        s1 = e1.sum(1, keepdim=True)
        lab = s["targets"] >= 0
        tgt = s["targets"].clamp(min=0).long()
        ce = (m + s1.log())[:, 0] - z[rows, tgt]
        loss = loss + hard * torch.where(lab, ce, 0.0)
        e1.div_(s1)
        e1[rows, tgt] -= 1.0
        grad.add_(e1 * (hard * lab.float())[:, None])
    row_loss = torch.where(w != 0, loss * w, 0.0)
    grad = torch.where(w[:, None] != 0, grad * (w * s["scale"])[:, None], 0.0)
    return {"row_loss": row_loss, "loss": row_loss.double().sum().float().reshape(1),
            "dlogits": grad.to(s["logits"].dtype)}


def _plain_select(s, c):
    # totals in 64 bits: two candidates may be nearer than 32 bits tell apart
    b, w, v = c["batch"], c["beams"], c["vocab"]
    x = _finite(s["logits"])
    k = min(w, v)
    top, idx = _top_rows(x, k)
    d = x.double()
    m = d.amax(1, keepdim=True)
    m = torch.where(m > -INF, m, 0.0)
    lse = m + (d - m).exp().sum(1, keepdim=True).log()
    score = s["scores"].double()[:, None]
    total = torch.where(top > -INF, score + (top.double() - lse), -INF)
    done = (s["finished"] != 0)[:, None]
    first = torch.arange(k, device=x.device)[None, :] == 0
    total = torch.where(done, torch.where(first, score, -INF), total)
    idx = torch.where(done, s["eos"], idx)
    total, at = total.reshape(b, w * k).sort(dim=1, descending=True, stable=True)
    total, at = total[:, :w], at[:, :w]
    live = total > -INF
    place = torch.arange(w, device=x.device)[None, :].expand(b, w)
    parents = torch.where(live, at // k, place)
    tokens = torch.where(live, idx.reshape(b, w * k).gather(1, at), s["eos"])
    was = (s["finished"] != 0).reshape(b, w).gather(1, parents)
    return {"scores": total.float().reshape(-1), "tokens": tokens.to(torch.int32).reshape(-1),
            "parents": parents.to(torch.int32).reshape(-1),
            "finished": (was | (tokens == s["eos"])).to(torch.int32).reshape(-1)}


def _plain_reorder(s, c):
    b, w, x = c["batch"], c["beams"], s["state"]
    at = (s["parents"].reshape(b, w) + w * torch.arange(b, device=x.device)[:, None]).reshape(-1)
    x.copy_(x.index_select(1, at.long()))
    return {"state": x}


def _plain_backtrack(s, c):
    t, b, w = c["steps"], c["batch"], c["beams"]
    # row i of `at`: which beam of step i the last step's beams descend from;
    # the maps are composed over doubling distances
    at = torch.empty(t, b, w, device="cuda", dtype=torch.int64)
    at[-1] = torch.arange(w, device="cuda")
    at[:-1] = s["parents"].reshape(t, b, w)[1:]
    step = 1
    while step < t:
        at[:t - step] = at[:t - step].gather(2, at[step:].clone())
        step *= 2
    seq = s["tokens"].reshape(t, b, w).gather(2, at).permute(1, 2, 0)
    ended = (seq == s["eos"]).to(torch.int32).cumsum(2)
    lengths = (t - (ended > 0).sum(2)).clamp(max=t - 1) + 1
    seq = torch.where(ended > 0, s["eos"], seq)
    score = s["scores"].double().reshape(b, w) / lengths.double().pow(ALPHA)
    score, order = score.sort(dim=1, descending=True, stable=True)
    seq = seq.gather(1, order[:, :, None].expand(b, w, t))
    return {"sequences": seq.reshape(b * w, t).to(torch.int32),
            "lengths": lengths.gather(1, order).to(torch.int32).reshape(-1),
            "ranked": score.float().reshape(-1)}


_OWN = {"topk": _own_topk, "distill": _own_distill, "select": _own_select,
        "reorder": _own_reorder, "backtrack": _own_backtrack}
_PLAIN = {"topk": _plain_topk, "distill": _plain_distill, "select": _plain_select,
          "reorder": _plain_reorder, "backtrack": _plain_backtrack}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "topk":
        return {"top": s["logits"].double().sort(dim=1, descending=True)[0][:, :c["k"]],
                "idx": None, "lse": torch.logsumexp(s["logits"].double() / c["tau"], 1)}
    if c["op"] == "distill":
        return _exact_distill(s, c)
    if c["op"] == "select":
        b, w, v = c["batch"], c["beams"], c["vocab"]
        t = torch.log_softmax(s["logits"].double(), 1) + s["scores"].double()[:, None]
        done = s["finished"] != 0
        t[done] = -INF
        t[done, s["eos"]] = s["scores"].double()[done]
        t = t.reshape(b, w * v).sort(dim=1, descending=True)[0][:, :w]
        return {"scores": t.reshape(-1), "tokens": None, "parents": None, "finished": None}
    if c["op"] == "reorder":
        return None
    t, b, w = c["steps"], c["batch"], c["beams"]
    tok, par = s["tokens"].cpu().reshape(t, b, w), s["parents"].cpu().reshape(t, b, w).long()
    at = torch.arange(w).expand(b, w)
    length = torch.full((b, w), t)
    for i in range(t - 1, -1, -1):
        length = torch.where(tok[i].gather(1, at) == s["eos"], i + 1, length)
        at = par[i].gather(1, at)
    ranked = s["scores"].cpu().double().reshape(b, w) / length.double() ** ALPHA
    return {"sequences": None, "lengths": None,
            "ranked": ranked.sort(dim=1, descending=True)[0].reshape(-1)}


def _exact_distill(s, c):
    """The loss in 64 bits, and its gradient by automatic differentiation."""
    tau, hard, w = c["tau"], c["hard"], s["weight"].double()
    z = s["logits"].double().requires_grad_()
    has = s["idx"] >= 0
    at = s["idx"].clamp(min=0).long()
    logp = torch.log_softmax(torch.where(has, s["top"].double() / tau, -INF), 1)
    logp = torch.where(has, logp, 0.0)
    logq = torch.log_softmax(z / tau, 1).gather(1, at)
    kl = torch.where(has, logp.exp() * (logp - logq), 0.0).sum(1)
    loss = (1.0 - hard) * tau * tau * kl
    if hard:
        lab = s["targets"] >= 0
        ce = -torch.log_softmax(z, 1).gather(1, s["targets"].clamp(min=0).long()[:, None])[:, 0]
        loss = loss + hard * torch.where(lab, ce, 0.0)
    loss = loss * w
    total = loss.sum()
    grad, = torch.autograd.grad(total * s["scale"], z)
    return {"row_loss": loss.detach(), "loss": total.detach().reshape(1), "dlogits": grad}
