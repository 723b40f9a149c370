"""logits_process where a row's tokens are shared out in other runs: one wave
of CTAs by 1 to 5 spans each, more than one wave, more rows than a wave."""
import pytest
import torch

from molten_b200 import sample
from tests.test_logits_rules_gpu import case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,V,f32,biased", [
    (48, 128000, False, 300), (64, 128000, False, 300), (64, 128000, False, 0), (56, 128001, False, 3), (58, 127999, True, 40),
    (100, 65536, True, 20), (130, 65537, False, 1), (800, 4097, False, 5), (800, 9000, True, 0), (1500, 300, False, 2)])
def test_rules_over_waves(cuda_ctx, B, V, f32, biased):
    x, r, d = case(B + V, B, V, f32, biased=biased, mask="own")
    out, best = torch.full_like(x, float("nan")), torch.zeros(B, dtype=torch.int64, device="cuda")
    sample.logits_process(cuda_ctx, x, out, r, best)
    check(out, x, r, d, best, cuda_ctx)
