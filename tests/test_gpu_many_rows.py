"""Calls of so many rows that a launch of a thread, or a few, for each would pass 2^32 threads
(such a launch runs their number modulo 2^32, without an error)."""
import pytest

pytestmark = pytest.mark.gpu


def room(n):
    import torch
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < n:
        pytest.skip("not enough memory free")


# 16 lanes a row, and a wave a row
@pytest.mark.parametrize("rows,experts,top_k", [(2 ** 28 + 5, 2, 1), (2 ** 26 + 3, 17, 16)])
def test_routing(smg, rows, experts, top_k):
    import torch
    room(20 << 30)
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.empty(rows, experts, dtype=torch.float16, device="cuda").normal_(generator=g)
    ids = torch.full((rows, top_k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((rows, top_k), -7.0, device="cuda")
    smg.Router(experts, top_k).route(logits, None, ids, w, rows)
    assert int(ids.min()) >= 0 and float(w.min()) >= 0
    for at in (0, rows // 2, rows - 1000):
        l = logits[at:at + 1000].float()
        want = torch.sort(l, dim=1, descending=True, stable=True)
        assert torch.equal(ids[at:at + 1000], want.indices[:, :top_k].int())
        assert torch.allclose(w[at:at + 1000], torch.softmax(want.values[:, :top_k], 1), rtol=1e-5, atol=0)
