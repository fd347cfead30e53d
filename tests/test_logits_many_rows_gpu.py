"""As many rows as an int counts (rows of one logit, about 36 GB), and the longest row."""
import math

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture
def room(cuda):
    cuda.cuda.empty_cache()
    if cuda.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of free device memory")
    yield cuda
    cuda.cuda.empty_cache()


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 5000])
def test_distillation(rnet, room, n):
    """One logit has the probability 1 whatever it is: with the teacher's normaliser the
    row's loss is p log p, p = exp(t - lse)."""
    torch = room
    z = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    idx = torch.zeros(n, dtype=torch.int32, device="cuda")
    t = torch.ones(n, device="cuda")
    lse = torch.full((n,), 0.5, device="cuda")
    row, loss = torch.full((n,), 9.0, device="cuda"), torch.zeros(1, device="cuda")
    rnet.call("rnet_distill_topk_forward", z.data_ptr(), rnet.DTYPE_BF16, 1, idx.data_ptr(),
              t.data_ptr(), lse.data_ptr(), None, None, 1.0, 1.0, 0.0, 1.0, row.data_ptr(),
              loss.data_ptr(), None, 0, n, 1, 1, None)
    torch.cuda.synchronize()
    del z, idx, t, lse
    one = 0.5 * math.exp(0.5)
    assert torch.all((row >= one * (1 - 16 * U)) & (row <= one * (1 + 16 * U)))
    assert abs(float(loss) - n * one) <= 17 * U * n * one


def test_records(rnet, room):
    torch, n = room, 2 ** 31 - 1
    z = torch.full((n,), 1.5, dtype=torch.bfloat16, device="cuda")
    z[n - 1] = 2.0
    idx = torch.full((n,), 7, dtype=torch.int32, device="cuda")
    top = torch.full((n,), 7.0, device="cuda")
    rnet.call("rnet_topk_logits_forward", z.data_ptr(), rnet.DTYPE_BF16, 1, 1.0, top.data_ptr(),
              idx.data_ptr(), None, n, 1, 1, None)
    torch.cuda.synchronize()
    assert torch.all(idx == 0) and torch.all(top[:n - 1] == 1.5) and float(top[n - 1]) == 2.0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_largest_vocabulary(rnet, room, dtype):
    """A row of 2^30 logits. A thread adds a partial sum for each of 65536 chunks."""
    torch, v, k = room, 1 << 30, 64
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    z = torch.full((v,), -2.0, dtype=t, device="cuda")
    at = [v - 1, 0, v // 2, v // 2 - 1, 12345, v - 12345] + [(i * v) // 59 + 7 for i in range(58)]
    for i, a in enumerate(at):
        z[a] = 18.0 - i / 8
    lse = torch.zeros(1, device="cuda")
    top, idx = torch.zeros(k, device="cuda"), torch.zeros(k, dtype=torch.int32, device="cuda")
    rnet.call("rnet_topk_logits_forward", z.data_ptr(), int(dtype == "bf16"), v, 1.0,
              top.data_ptr(), idx.data_ptr(), lse.data_ptr(), 1, v, k, None)
    s, out = torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda")
    tok, par = (torch.full((1,), 9, dtype=torch.int32, device="cuda") for _ in range(2))
    rnet.call("rnet_beam_select", z.data_ptr(), int(dtype == "bf16"), v, s.data_ptr(), None, -1,
              out.data_ptr(), tok.data_ptr(), par.data_ptr(), None, 1, 1, v, None)
    assert rnet.device_error(clear=True) == 0
    assert idx.tolist() == at and top.tolist() == [18.0 - i / 8 for i in range(64)]
    want = math.log(sum(math.exp(18.0 - i / 8) for i in range(64)) + (v - 64) * math.exp(-2.0))
    assert abs(float(lse) - want) <= (2 * 65536 + 200) * U
    assert tok.tolist() == [v - 1] and par.tolist() == [0]
    assert abs(float(out) - (18.0 - want)) <= (2 * 65536 + 200) * U
