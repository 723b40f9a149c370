"""What the serving entry points say to arguments that share memory (as
tests/test_serving_cpu.py: no GPU, made-up addresses)."""
import pytest

from molten_b200 import _lib
from tests.test_serving_cpu import answer, lib  # noqa: F401

PAGE = 8 * 16 * 64  # elements of a page of 8 KV heads x 16 tokens x 64, at 2 bytes


@pytest.mark.parametrize("changed", [
    dict(v_cache=0x100000),                                                 # one cache for both
    dict(v_cache=0x100000 + 2 * PAGE),                                      # a page further
    dict(v_cache=0x100000 + 2 * 7 * PAGE),                                  # V's first page is K's last
    dict(v_cache=0x100000 + 2 * PAGE - 16, block_stride=2 * PAGE),          # the halves of one tensor, 16 bytes short
    dict(k_cache=0x100000 + 2 * PAGE - 16, v_cache=0x100000, block_stride=2 * PAGE),
    dict(v_cache=0x100000 + 2 * 3 * PAGE + 16, block_stride=2 * PAGE),
    dict(v_cache=0x100000, kv_dtype=_lib.DTYPE_E4M3),
    dict(v_cache=0x100000 + 2 * PAGE - 16, num_blocks=1),
])
def test_k_and_v_written_to_the_same_rows_are_refused(lib, changed):  # noqa: F811
    rc, why = answer(lib, "mc_qk_norm_rope", **changed)
    assert rc == _lib.MC_EINVAL and "k_cache overlaps v_cache" in why, why


@pytest.mark.parametrize("changed", [
    dict(v_cache=0x100000, v=None),                                         # only K is written
    dict(v_cache=0x100000 + 2 * PAGE, block_stride=2 * PAGE),               # the halves of one tensor
    dict(k_cache=0x100000 + 2 * PAGE, v_cache=0x100000, block_stride=2 * PAGE),
    dict(v_cache=0x100000 + PAGE, block_stride=2 * PAGE, kv_dtype=_lib.DTYPE_E4M3),
    dict(v_cache=0x100000 + 2 * 3 * PAGE, block_stride=2 * PAGE),           # in the gaps, a page further
    dict(v_cache=0x100000 + 2 * 8 * PAGE),                                  # behind the last page
    dict(v_cache=0x100000 + 2 * PAGE, num_blocks=1),
])
def test_k_and_v_beside_each_other_reach_the_context(lib, changed):  # noqa: F811
    rc, why = answer(lib, "mc_qk_norm_rope", **changed)
    assert rc == _lib.MC_EINVAL and "null context" in why, why


def test_attention_may_read_one_cache_as_k_and_v(lib):  # noqa: F811
    rc, why = answer(lib, "mc_paged_attention", v_cache=0x100000)
    assert rc == _lib.MC_EINVAL and "null context" in why, why
