"""The gated scan and its step at their limits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_step_of_nearly_all_elements_that_32_bits_count():
    import snntc_amd as snn
    torch.cuda.empty_cache()
    n = 2 ** 32 - 100
    if torch.cuda.mem_get_info()[0] < 10 * n + (4 << 30):
        pytest.skip("needs 45 GB of the card's memory")
    x = torch.ones(n, device=DEV)
    gate = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    x[-5:] = 3.0
    out = snn.gated_step(x, gate)
    assert (out[-5:] == 1.5).all()
    out[-5:] = 0.5
    assert all((part == 0.5).all() for part in out.split(2 ** 29))
