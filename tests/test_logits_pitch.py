"""Row pitches whose byte offsets cannot be counted: refused by every operator on rows of
logits, with no launch. Needs no GPU."""
import pytest

FAR = 0x7f0000000000  # an address; nothing is read


@pytest.mark.parametrize("ld", [2 ** 60, 2 ** 61, 2 ** 63 - 1])
@pytest.mark.parametrize("name,args", [
    ("rnet_topk_logits_forward", lambda ld: (FAR, 0, ld, 1.0, FAR, FAR, None, 2, 8, 2, None)),
    ("rnet_distill_topk_forward", lambda ld: (FAR, 0, ld, FAR, FAR, None, None, None, 1.0, 1.0,
                                              0.0, 1.0, FAR, None, None, 0, 2, 8, 2, None)),
    ("rnet_beam_select", lambda ld: (FAR, 1, ld, FAR, None, -1, FAR, FAR, FAR, None, 1, 2, 8,
                                     None))])
def test_refused(rnet, name, args, ld):
    n0 = rnet.kernel_launches()
    with pytest.raises(rnet.RnetError, match="row pitch too large"):
        rnet.call(name, *args(ld))
    assert rnet.kernel_launches() == n0
