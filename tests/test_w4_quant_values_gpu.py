"""The 4-bit quantiser at weights that are no numbers and at the ends of their types."""
import pytest
import torch

from dlblas_amd.kernels.w4_gemm import per_group_quant_w4, w4_gemm
from oracle import decoder as orc

pytestmark = pytest.mark.gpu
bf16, f16 = torch.bfloat16, torch.float16


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def on(dev, *tensors):
    return [None if t is None else t.to(dev) for t in tensors]


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('zero_points', [False, True])
@pytest.mark.parametrize('group', [32, 64, 128])
@pytest.mark.parametrize('bad', ['nan', '-nan', 'inf', '-inf'])
def test_a_weight_that_is_no_number_shows(dev, bad, group, zero_points, dtype):
    """Its whole group dequantises to NaN; the other groups are what they are without it."""
    w = torch.randn(6, 512, generator=torch.Generator().manual_seed(3)).to(dtype)
    value = -torch.tensor(float('nan')) if bad == '-nan' else torch.tensor(float(bad))
    places = [(0, 0), (1, group - 1), (2, 511), (4, 200), (4, 201)]
    poor = w.clone()
    hit = torch.zeros(6, 512 // group, dtype=torch.bool)
    for r, c in places:
        poor[r, c] = value
        hit[r, c // group] = True
    poor[5, :group] = value  # nothing but such values
    hit[5, 0] = True
    q, s, z = (None if t is None else t.cpu() for t in per_group_quant_w4(poor.to(dev), group, zero_points))
    clean = [None if t is None else t.cpu() for t in per_group_quant_w4(w.to(dev), group, zero_points)]
    back = orc.w4_weights(q, s, z).reshape(6, -1, group)
    assert bool(back[hit].isnan().all())
    assert torch.equal(back[~hit], orc.w4_weights(*clean).reshape(6, -1, group)[~hit])
    y = w4_gemm(torch.ones(2, 512, dtype=dtype, device=dev), *on(dev, q, s, z)).cpu()
    assert torch.equal(y.isnan(), hit.any(1)[None].expand(2, 6))


@pytest.mark.parametrize('zero_points', [False, True])
def test_weights_at_the_ends_of_their_type(dev, zero_points):
    """The largest finite numbers are numbers; a range from lowest to highest that fp32 does not hold is none."""
    top = torch.finfo(f16).max
    w = torch.tensor([[top, -top] * 16, [top] * 32, [-top] * 32]).to(f16)
    q, s, z = (None if t is None else t.cpu() for t in per_group_quant_w4(w.to(dev), 32, zero_points))
    back = orc.w4_weights(q, s, z)
    assert float((back - w.double()).abs().max()) <= float(s.double().max())
    top = torch.finfo(bf16).max
    w = torch.tensor([[top, -top] * 16, [top] * 32, [-top] * 32]).to(bf16)
    q, s, z = (None if t is None else t.cpu() for t in per_group_quant_w4(w.to(dev), 32, zero_points))
    back = orc.w4_weights(q, s, z)
    assert float((back[1:] - w[1:].double()).abs().max()) <= float(s[1:].double().max())
    assert bool(back[0].isnan().all()) if zero_points else float((back[0] - w[0].double()).abs().max()) <= float(s[0].double().max())
