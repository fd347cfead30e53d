"""The decoder's beam search and the training step on a teacher's records: the
operators on logits and beams as the model runs them.

The search's oracle runs the CPU oracle's full-sequence forward on every beam at
every step and keeps whole token lists. Its candidates must lie further apart than
GAP, which is above what the decode path's logits may differ by (1e-4 of the
largest logit is the decode parity tolerance; the measured difference at this size
is below 1e-5)."""
import ctypes

import numpy as np
import pytest

import logits_oracle as ref

pytestmark = pytest.mark.gpu

GAP = 2e-5
D, L, F, S, V, T = 64, 2, 128, 160, 256, 20
BATCH, BEAMS, STEPS = 3, 4, 7
SEED, SCALE = 6, 12.0


def params_and_prompts(rnet, rdata):
    cfg = rnet.ModelConfig.make(d_model=D, n_layers=L, d_ff=F, n_slots=S, top_k=2, vocab=V,
                                seq_len=T + STEPS + 4)
    p = rdata.init_params_normal(cfg, seed=SEED, std=0.05)
    rdata.split(cfg, p)["output"][:] *= SCALE  # logits that are not all alike
    prompts = np.random.default_rng(SEED).integers(0, V, size=(BATCH, T)).astype(np.int32)
    return cfg, p, prompts


def oracle_search(orc, params, prompts, beams, steps, eos, alpha):
    """Per sequence: ranked [(score, tokens, length)], and the smallest gap met."""
    ocfg = orc.make_config(D, L, F, S, 2, V, seq_len=T + STEPS + 4)
    out, gap = [], np.inf
    for prompt in prompts:
        live = [(0.0, [], False)]
        for _ in range(steps):
            n = len(live[0][1])
            seqs = np.array([list(prompt) + t for _, t, _ in live], np.int32)
            lg, _, _ = orc.forward(ocfg, params, np.ascontiguousarray(seqs), len(live), T + n)
            lp = lg.reshape(len(live), T + n, V)[:, -1].astype(np.float64)
            lp = lp - ref.logsumexp(lp)[:, None]
            new = []
            for i, (s, t, done) in enumerate(live):
                if done:
                    new.append((s, i, eos, t, True))
                else:
                    new += [(s + lp[i, w], i, w, t, w == eos) for w in range(V)]
            new.sort(key=lambda c: (-c[0], c[1], c[2]))
            gap = min(gap, min(-np.diff([c[0] for c in new[:beams + 1]])))
            live = [(s, t + [w], done) for s, _, w, t, done in new[:beams]]
        rows = []
        for s, t, _ in live:
            k = t.index(eos) + 1 if eos in t else steps
            rows.append((s / float(k) ** alpha, t, k))
        order = sorted(range(beams), key=lambda j: (-rows[j][0], j))
        gap = min(gap, min(-np.diff([rows[j][0] for j in order])))
        out.append([rows[j] for j in order])
    return out, gap


def _decoder(rnet, torch, cfg, p, prompts, beams):
    m = rnet.Model(cfg, device=0, reference_init=False)
    m.set_params(p)
    dec = rnet.Decoder(m, len(prompts) * beams)
    dec.prefill_beams(torch.from_numpy(prompts.reshape(-1)).cuda(), prompts.shape[1], beams)
    return m, dec


def _search(torch, m, dec, beams, steps, **kw):
    seq = torch.full((dec.M, steps), -9, dtype=torch.int32, device="cuda")
    ln = torch.full((dec.M,), -9, dtype=torch.int32, device="cuda")
    sc = torch.full((dec.M,), 9.0, device="cuda")
    dec.beam_search(beams, steps, seq, ln, sc, **kw)
    m.synchronize()
    return seq.cpu().numpy(), ln.cpu().numpy(), sc.cpu().numpy()


# eos = 10: a token that beams of this model choose, so that some end early
@pytest.mark.parametrize("eos,alpha", [(-1, 0.0), (10, 0.0), (10, 0.9)])
@pytest.mark.parametrize("graph", [False, True])
def test_beam_search_matches_the_oracle(rnet, rdata, orc, cuda, eos, alpha, graph):
    torch = cuda
    cfg, p, prompts = params_and_prompts(rnet, rdata)
    want, gap = oracle_search(orc, p, prompts, BEAMS, STEPS, eos, alpha)
    assert gap > GAP, "the input's candidates lie too close together"
    m, dec = _decoder(rnet, torch, cfg, p, prompts, BEAMS)
    seq, ln, sc = _search(torch, m, dec, BEAMS, STEPS, eos=eos, length_alpha=alpha,
                          use_graph=graph)
    for g, rows in enumerate(want):
        for j, (s, t, n) in enumerate(rows):
            i = g * BEAMS + j
            assert list(seq[i]) == t and ln[i] == n
            assert abs(sc[i] - s) <= 1e-4 * abs(s)
    dec.close()
    m.close()


def test_one_beam_is_greedy_and_searches_repeat(rnet, rdata, cuda):
    """beams = 1 gives the greedy tokens; a second search after another prefill, of
    another length and eos, gives what a new decoder gives; prefilling every
    stream with its prompt equals prefill_beams."""
    torch = cuda
    cfg, p, prompts = params_and_prompts(rnet, rdata)
    m, dec = _decoder(rnet, torch, cfg, p, prompts, 1)
    seq, ln, _ = _search(torch, m, dec, 1, STEPS)
    dec.prefill(torch.from_numpy(prompts.reshape(-1)).cuda(), T)
    _, first = dec.outputs_host()
    out = torch.zeros(STEPS - 1, dec.M, dtype=torch.int32, device="cuda")
    dec.generate(STEPS - 1, out)
    m.synchronize()
    greedy = np.concatenate([first[:, None], out.cpu().numpy().T], axis=1)
    np.testing.assert_array_equal(seq, greedy)
    assert np.all(ln == STEPS)
    dec.close()
    m.close()

    m, dec = _decoder(rnet, torch, cfg, p, prompts, BEAMS)
    a = _search(torch, m, dec, BEAMS, STEPS, eos=10, length_alpha=0.5)
    dec.prefill(torch.from_numpy(np.repeat(prompts, BEAMS, 0).reshape(-1)).cuda(), T)
    b = _search(torch, m, dec, BEAMS, STEPS + 3, eos=-1)
    dec.prefill_beams(torch.from_numpy(prompts.reshape(-1)).cuda(), T, BEAMS)
    c = _search(torch, m, dec, BEAMS, STEPS, eos=10, length_alpha=0.5)
    for x, y in zip(a, c):
        np.testing.assert_array_equal(x, y)
    dec.close()
    m.close()
    m, dec = _decoder(rnet, torch, cfg, p, prompts, BEAMS)
    d = _search(torch, m, dec, BEAMS, STEPS + 3, eos=-1, use_graph=False)
    for x, y in zip(b, d):
        np.testing.assert_array_equal(x, y)
    dec.close()
    m.close()


def test_a_search_of_one_step(rnet, rdata, cuda):
    """The best tokens of each prompt, by the logits of the prefill."""
    torch = cuda
    cfg, p, prompts = params_and_prompts(rnet, rdata)
    m, dec = _decoder(rnet, torch, cfg, p, prompts, BEAMS)
    lg, _ = dec.outputs_host()
    seq, ln, sc = _search(torch, m, dec, BEAMS, 1)
    for g in range(BATCH):
        x = lg[g * BEAMS].astype(np.float64)
        best = np.argsort(-x, kind="stable")[:BEAMS]
        rows = slice(g * BEAMS, (g + 1) * BEAMS)
        np.testing.assert_array_equal(seq[rows, 0], best)
        lp = x[best] - ref.logsumexp(x)
        assert np.all(np.abs(sc[rows] - lp) <= ref.lse_bound(lp, V) + np.abs(lp) * ref.U)
    assert np.all(ln == 1)
    dec.close()
    m.close()


def test_the_streams_hold_the_beams_afterwards(rnet, rdata, orc, cuda):
    """step(None) after a search feeds the last tokens: the logits are those of the
    whole sequences (with length_alpha 0 the ranking is the streams' order)."""
    torch = cuda
    cfg, p, prompts = params_and_prompts(rnet, rdata)
    m, dec = _decoder(rnet, torch, cfg, p, prompts, BEAMS)
    seq, _, _ = _search(torch, m, dec, BEAMS, STEPS)
    dec.step(None)
    lg, _ = dec.outputs_host()
    full = np.concatenate([np.repeat(prompts, BEAMS, 0), seq], axis=1).astype(np.int32)
    ocfg = orc.make_config(D, L, F, S, 2, V, seq_len=T + STEPS + 4)
    want, _, _ = orc.forward(ocfg, p, np.ascontiguousarray(full), len(full), T + STEPS)
    want = want.reshape(len(full), T + STEPS, V)[:, -1]
    assert np.abs(lg - want).max() <= 1e-4 * np.abs(want).max()
    dec.close()
    m.close()


def test_beam_search_refusals(rnet, rdata, cuda):
    torch = cuda
    cfg, p, prompts = params_and_prompts(rnet, rdata)
    m, dec = _decoder(rnet, torch, cfg, p, prompts, BEAMS)
    tok = torch.from_numpy(prompts.reshape(-1)).cuda()
    seq = torch.full((dec.M, 4), -9, dtype=torch.int32, device="cuda")
    ln, sc = torch.full((dec.M,), -9, dtype=torch.int32, device="cuda"), torch.ones(dec.M).cuda()
    n0 = rnet.kernel_launches()
    for beams, steps, kw, text in [(5, 4, {}, "multiple of beams"), (33, 4, {}, "beams must be"),
                                   (0, 4, {}, "beams must be"), (4, 0, {}, "n_steps"),
                                   (4, 4, dict(eos=V), "eos"), (4, 4, dict(eos=-2), "eos"),
                                   (4, 4, dict(length_alpha=float("nan")), "finite")]:
        with pytest.raises(rnet.RnetError, match=text):
            dec.beam_search(beams, steps, seq, ln, sc, **kw)
    with pytest.raises(rnet.RnetError, match="null"):
        dec.beam_search(4, 4, None, ln, sc)
    for beams in (0, 5):
        with pytest.raises(rnet.RnetError, match="multiple of beams"):
            dec.prefill_beams(tok, T, beams)
    assert rnet.kernel_launches() == n0
    m.synchronize()
    assert torch.all(seq == -9) and torch.all(ln == -9) and torch.all(sc == 1)
    dec.close()
    m.close()


# ------------------------------------------------------------------ training
def _pair(rnet, rdata, seed):
    cfg = rnet.ModelConfig.make(d_model=D, n_layers=L, d_ff=F, n_slots=S, top_k=2, vocab=V,
                                seq_len=48)
    m = rnet.Model(cfg, device=0, reference_init=False)
    p = rdata.init_params_normal(cfg, seed=seed, std=0.05)
    m.set_params(p)
    return m, p


def test_step_on_hard_labels_alone_is_the_training_step(rnet, rdata, cuda):
    """soft_weight 0, hard_weight 1: the loss is the cross-entropy. The two kernels
    round differently: the gradients agree to 1e-5 of their norm, the summed loss
    (terms of about log 256, a few roundings each) to 1e-6."""
    torch = cuda
    B, N = 3, 3 * 40
    r = np.random.default_rng(3)
    tok = torch.from_numpy(r.integers(0, V, size=N).astype(np.int32)).cuda()
    tgt = torch.from_numpy(r.integers(0, V, size=N).astype(np.int32)).cuda()
    idx = torch.zeros(N, 2, dtype=torch.int32, device="cuda")
    val = torch.zeros(N, 2, device="cuda")
    la, lb = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda")
    a, p = _pair(rnet, rdata, 1)
    b, _ = _pair(rnet, rdata, 1)
    a.train_step(tok, tgt, B, 40, 1e-2, 1.0, la)
    b.train_step_distill(tok, idx, val, B, 40, 2, soft_weight=0.0, hard_weight=1.0, d_tgt=tgt,
                         lr=1e-2, clip=1.0, d_loss_sum=lb)
    a.synchronize()
    b.synchronize()
    ga, gb = a.get_grads().astype(np.float64), b.get_grads().astype(np.float64)
    assert np.linalg.norm(ga - gb) <= 1e-5 * np.linalg.norm(ga)
    assert abs(float(la) - float(lb)) <= 1e-6 * abs(float(la))
    ua, ub = a.get_params() - p, b.get_params() - p
    assert np.linalg.norm(ua - ub) <= 1e-4 * np.linalg.norm(ua)
    a.close()
    b.close()


@pytest.mark.parametrize("bf16", [False, True])
def test_a_student_trains_on_a_teachers_records(rnet, rdata, cuda, bf16):
    """Teacher forward, its records, two student steps. Each step equals forward,
    rnet_distill_topk_forward, backward and step by hand (bit for bit: the same
    launches), and its loss is the 64-bit loss of the student's logits."""
    torch = cuda
    B, TT, K, tau = 4, 40, 12, 2.0
    N = B * TT
    r = np.random.default_rng(7)
    tok = torch.from_numpy(r.integers(0, V, size=N).astype(np.int32)).cuda()
    tgt_h = r.integers(0, V, size=N).astype(np.int32)
    tgt_h[::7] = -1
    w_h = np.where(np.arange(N) % TT >= TT - 5, 0.0, 1.0).astype(np.float32)  # padded ends
    tgt, w = torch.from_numpy(tgt_h).cuda(), torch.from_numpy(w_h).cuda()
    teacher, _ = _pair(rnet, rdata, 2)
    lg = torch.zeros(N, V, device="cuda")
    teacher.forward(tok, lg, B, TT)
    teacher.synchronize()
    lg *= 20.0  # a teacher with opinions
    val, lse = torch.zeros(N, K, device="cuda"), torch.zeros(N, device="cuda")
    idx = torch.zeros(N, K, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    stream = ctypes.c_void_p(teacher.stream())
    rnet.call("rnet_topk_logits_forward", lg.data_ptr(), 0, V, tau, val.data_ptr(),
              idx.data_ptr(), lse.data_ptr(), N, V, K, stream)
    teacher.synchronize()
    a, _ = _pair(rnet, rdata, 1)
    b, _ = _pair(rnet, rdata, 1)
    for m in (a, b):
        m.set_precision(bf16)
    z, dz = torch.zeros(N, V, device="cuda"), torch.zeros(N, V, device="cuda")
    row, loss, by_hand = (torch.zeros(n, device="cuda") for n in (N, 1, 1))
    for _ in range(2):
        a.train_step_distill(tok, idx, val, B, TT, K, tau, 0.75, 0.25, d_tgt=tgt,
                             d_teacher_lse=lse, d_row_weight=w, lr=1e-2, clip=1.0,
                             d_loss_sum=loss)
        b.zero_grad()
        b.forward(tok, z, B, TT)
        rnet.call("rnet_distill_topk_forward", z.data_ptr(), 0, V, idx.data_ptr(), val.data_ptr(),
                  lse.data_ptr(), tgt.data_ptr(), w.data_ptr(), tau, 0.75, 0.25, 1.0 / N,
                  row.data_ptr(), by_hand.data_ptr(), dz.data_ptr(), V, N, V, K,
                  ctypes.c_void_p(b.stream()))
        b.backward(dz, tok, B, TT)
        b.step(1e-2, 1.0)
        a.synchronize()
        b.synchronize()
        assert float(loss) == float(by_hand)
        l0, g0, bl, bg = ref.distill(z.cpu().numpy(), idx.cpu().numpy(), val.cpu().numpy(), tau,
                                     0.75, 0.25, 1.0 / N, t_lse=lse.cpu().numpy(), targets=tgt_h,
                                     weight=w_h)
        assert abs(float(loss) - l0.sum()) <= bl.sum() + abs(l0.sum()) * ref.U
        assert np.all(np.abs(dz.cpu().numpy() - g0) <= bg + 1e-38)
        ga, gb = a.get_grads(), b.get_grads()
        # scatter gradients of the slots are summed by atomics: not bit for bit
        assert np.linalg.norm(ga - gb) <= 1e-5 * np.linalg.norm(gb)
    for m in (a, b, teacher):
        m.close()


def test_distill_step_refusals(rnet, rdata, cuda):
    torch = cuda
    m, p = _pair(rnet, rdata, 1)
    tok = torch.zeros(32, dtype=torch.int32, device="cuda")
    idx, val = torch.zeros(32, 2, dtype=torch.int32, device="cuda"), torch.zeros(32, 2).cuda()
    n0 = rnet.kernel_launches()
    for args, kw, text in [((None, idx, val, 1, 32, 2), {}, "null"),
                           ((tok, None, val, 1, 32, 2), {}, "null"),
                           ((tok, idx, val, 0, 32, 2), {}, "seq_len"),
                           ((tok, idx, val, 65, 48, 2), {}, "seq_len"),
                           ((tok, idx, val, 1 << 20, 1 << 14, 2), {}, "seq_len"),
                           ((tok, idx, val, 1, 32, 65), {}, "top_k"),
                           ((tok, idx, val, 1, 32, 2), dict(temperature=0.0), "temperature"),
                           ((tok, idx, val, 1, 32, 2), dict(soft_weight=float("nan")), "finite"),
                           ((tok, idx, val, 1, 32, 2), dict(hard_weight=0.5), "targets")]:
        with pytest.raises(rnet.RnetError, match=text):
            m.train_step_distill(*args, **kw)
    assert rnet.kernel_launches() == n0
    np.testing.assert_array_equal(m.get_params(), p)
    m.close()
