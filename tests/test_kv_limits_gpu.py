"""The paged attention at its limits: a wait that only a part of a warp runs
out of, weights far below the largest one."""
import math

import pytest
import torch

from molten_b200 import _lib, kv
from tests import serving_ref as ref
from tests.test_kv_gpu import attention_case, check_attention, gen, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,H,K,fp8", [(64, 8, 2, False), (128, 8, 2, False), (64, 32, 2, True), (128, 8, 2, True)])
def test_a_wait_that_one_lane_runs_out_of(cuda_ctx, D, H, K, fp8):
    """One lane gives up just before the copies are reported, the other 31 find
    them: the warp gives up as one. The status says so, what it was working on
    is NaN, everything else is right, and the next call is whole again."""
    lens = [6000, 3, 9000, 0, 700]
    q, cache, table, keys = attention_case(14, lens, H, K, D, 16, fp8)
    ws, st = kv.paged_attention_workspace(D), torch.zeros(1, dtype=torch.int32, device="cuda")
    out, n = torch.empty_like(q), i32(lens)
    kv.paged_attention(cuda_ctx, q, cache, table, n, out, ws, status=st)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    cuda_ctx.set_test_flags(_lib.TEST_LATE_KV_ARRIVE)
    try:
        begin.record()
        kv.paged_attention(cuda_ctx, q, cache, table, n, out, ws, status=st)
        end.record()
        torch.cuda.synchronize()
    finally:
        cuda_ctx.set_test_flags(0)
    assert begin.elapsed_time(end) < 500, "the other lanes' waits (1 s at most) found the copies"
    assert st.item() == _lib.KV_WAIT
    for r in range(len(lens)):
        k, v = keys[r]
        want, _, e, _ = ref.attention(q[r], k, v, D ** -0.5)
        right = (out[r].double() - want).abs() <= ref.BF16_HALF * want.abs() + 1.01 * e
        assert bool((right | torch.isnan(out[r])).all())
        assert bool(torch.isnan(out[r]).any()) == (r == 0)
    st.zero_()
    kv.paged_attention(cuda_ctx, q, cache, table, n, out, ws, status=st)
    check_attention(out, None, q, keys, lens)
    assert st.item() == 0 and not ws[:4096].any()
