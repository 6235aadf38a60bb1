"""GPU: the scoring / loss / embedding / 8-bit operators at the edges of what their entry points take."""
import pytest
import torch

pytestmark = pytest.mark.gpu
H = 2.0 ** -24                       # half a step of f32


@pytest.mark.parametrize("n", [40, 3000])
@pytest.mark.parametrize("pad", [-1, -2, -50, 0])
def test_padding_rows_counted_from_the_end(pad, n):
    """The padding row stays zero under a step, by the one-launch gradient and by the sorted one."""
    import multimodalsum_amd as mm
    ids = (torch.arange(n, device="cuda") * 7) % 50
    m = mm.ScaledEmbedding(50, 16, scale=2.0, padding_idx=pad)
    y = m(ids)
    assert (y[ids == pad % 50] == 0).all()
    y.sum().backward()
    want = 2.0 * torch.bincount(ids, minlength=50).float()
    want[pad] = 0.0
    assert torch.equal(m.weight.grad, want[:, None].expand(50, 16))
    assert torch.equal(mm.scaled_embedding_grad(torch.ones(n, 16, device="cuda"), ids, 50, 2.0, padding_idx=pad), m.weight.grad)
