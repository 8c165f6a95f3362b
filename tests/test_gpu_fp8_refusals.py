"""What the 8-bit calls say where they refuse."""

import pytest
import torch

import tuna_b200

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("z_type", [torch.float16, torch.bfloat16, torch.float32], ids=str)
def test_z_beside_results_in_32_bits(z_type):
    f, n, k = 32, 4, 64
    q, s = tuna_b200.fp8_quantize(torch.zeros(2 * f, k, device="cuda"), "square")
    x, h = torch.zeros(n, k, device="cuda", dtype=torch.float16), torch.zeros(n, f, device="cuda")
    with pytest.raises(TypeError, match="h must be torch.float16 or torch.bfloat16"):
        tuna_b200.fp8_gated(x, None, q, s, h, f, n, k, z=torch.zeros(n, 2 * f, device="cuda", dtype=z_type))


def test_a_range_of_tokens_in_codes_has_its_scales_copied():
    m, n, k = 48, 50, 1040
    q, s = tuna_b200.fp8_quantize(torch.randn(m, k, device="cuda"), "square")
    x, xs = tuna_b200.fp8_quantize(torch.randn(n, k, device="cuda"))
    whole, part = torch.empty(n, m, device="cuda"), torch.empty(20, m, device="cuda")
    tuna_b200.fp8_matmul(x, xs, q, s, whole, m, n, k)
    with pytest.raises(ValueError, match="contiguous"):
        tuna_b200.fp8_matmul(x[10:30], xs[:, 10:30], q, s, part, m, 20, k)
    tuna_b200.fp8_matmul(x[10:30], xs[:, 10:30].contiguous(), q, s, part, m, 20, k)
    torch.cuda.synchronize()
    assert torch.equal(part, whole[10:30])
