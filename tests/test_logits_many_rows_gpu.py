"""As many rows as an int counts. Rows of one logit: about 36 GB."""
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
