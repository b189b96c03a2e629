"""The results of clip_gradient_norm are tensors of their own: what becomes of one does not reach the others."""
import pytest
import torch

import mops_b200.torch as mt


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes", [[5, 1000, 1, 0, 257], [300] * 40])
def test_each_result_has_memory_of_its_own(dtype, sizes):
    gradients = [torch.full((n,), 1.0 + i, dtype=dtype, device="cuda") for i, n in enumerate(sizes)] + [torch.ones(6, 4, dtype=torch.float32, device="cuda").T]
    _, clipped = mt.clip_gradient_norm(gradients, 1e6)  # (as they are)
    for c, g in zip(clipped, gradients):
        assert torch.equal(c, g) and c.stride() == g.stride() and c.storage_offset() == 0
        assert c.untyped_storage().nbytes() == g.numel() * g.element_size()
    places = [c.untyped_storage().data_ptr() for c in clipped if c.numel()]
    assert len(set(places)) == len(places)
    for c, n in zip(clipped, sizes):
        c.resize_(n + 2000).fill_(-1.0)
        assert (c == -1.0).all() and c.numel() == n + 2000
    assert torch.equal(clipped[-1], gradients[-1])
    _, clipped = mt.clip_gradient_norm(gradients, 1e6)
    clipped[0].resize_(100000).fill_(-1.0)
    for c, g in zip(clipped[1:], gradients[1:]):
        assert torch.equal(c, g)


@pytest.mark.gpu
def test_results_on_another_stream_outlive_the_call():
    """Memory that is given back while another stream still uses it is not handed out again."""
    gradients = [torch.ones(100003, device="cuda") for _ in range(30)]
    _, clipped = mt.clip_gradient_norm(gradients, 1e6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        total = sum(c.sum() for c in clipped)
    for c in clipped:
        c.record_stream(side)
    del c, clipped
    others = [torch.full((100003,), -7.0, device="cuda") for _ in range(60)]
    torch.cuda.synchronize()
    assert float(total) == 30 * 100003 and len(others) == 60
