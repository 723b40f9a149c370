"""The serving entry points without a GPU: what each refuses (the C ABI checks
its arguments before it looks at the context, so a call that gets as far as
"null context" has passed them), the rotation table, and the split of the
attention's work over CTAs (tests/cpp/test_paged_split.cpp)."""
import ctypes as C
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from molten_b200 import _lib, build

ROOT = Path(__file__).resolve().parents[1]
INF = float("inf")


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


CACHE = dict(k_cache=0x100000, v_cache=0x200000, kv_dtype=_lib.DTYPE_BF16, num_blocks=8, block_size=16,
             block_stride=8 * 16 * 64)
# arguments in order; every pointer is a made-up aligned address that nothing reads
CALLS = {
    "mc_kv_plan": dict(lens=0x100, new_lens=0x200, n_req=4, block_size=16, block_table=0x300, table_width=8,
                       free_list=0x400, n_free=0x500, free_len=8, seq_lens=0x600, n_free_out=0x700, row_start=0x800,
                       positions=0x900, token_req=0xa00, kv_lens=0xb00, slots=0xc00, max_tokens=4, status=None),
    "mc_kv_release": dict(done=0x100, lens=0x200, n_req=4, block_size=16, block_table=0x300, table_width=8,
                          free_list=0x400, n_free=0x500, free_len=8, lens_out=0x600, n_free_out=0x700, status=None),
    "mc_qk_norm_rope": dict(q=0x1000000, q_stride=2048, k=0x2000000, k_stride=512,
                            v=0x3000000, v_stride=512, n_tokens=3, n_heads=32, n_kv_heads=8, head_dim=64,
                            q_norm_w=0x100, k_norm_w=0x200, eps=1e-5, positions=0x300, turns=0x400, rot_dim=64,
                            interleaved=0, q_out=0x4000000, q_out_stride=2048, slots=0x500, **CACHE, k_scale=None,
                            v_scale=None, status=None),
    "mc_paged_attention": dict(q=0x1000000, q_stride=2048, n_rows=4, n_heads=32, **CACHE, n_kv_heads=8, head_dim=64,
                               k_scale=None, v_scale=None, block_table=0x300, n_req=4, table_width=2, kv_lens=0x400,
                               row_req=None, window=0, scale=0.125, out=0x2000000, out_stride=2048, lse=None,
                               workspace=0x3000000, ws_bytes=1 << 26, status=None),
    "mc_logits_process": dict(logits=0x1000000, logits_stride=1000, dtype=_lib.DTYPE_BF16, vocab=1000, batch=2,
                              seen=0x100, counts=0x200, repetition=0x300, frequency=0x400, presence=0x500,
                              bias_start=0x600, bias_ids=0x700, bias_vals=0x800, n_bias=5, allowed=0x900,
                              allowed_row=None, n_allowed=2, out=0x2000000, out_stride=1000, keys=0xa00),
    "mc_logits_mark": dict(tokens=0x100, batch=2, seen=0x200, counts=0x300, vocab=1000),
}


def answer(lib, name, **changed):
    args = dict(CALLS[name])
    assert set(changed) <= set(args), set(changed) - set(args)
    rc = getattr(lib, name)(None, *{**args, **changed}.values())
    return rc, lib.mc_last_error().decode()


@pytest.mark.parametrize("name", sorted(CALLS))
def test_good_arguments_reach_the_context(lib, name):
    rc, why = answer(lib, name)
    assert rc == _lib.MC_EINVAL and "null context" in why, why


REFUSED = [
    ("mc_kv_plan", dict(n_req=0), "n_req"),
    ("mc_kv_plan", dict(block_size=0), "block size"),
    ("mc_kv_plan", dict(table_width=0), "table width"),
    ("mc_kv_plan", dict(free_len=0), "free list of 0"),
    ("mc_kv_plan", dict(max_tokens=0), "max_tokens"),
    ("mc_kv_plan", dict(lens=None), "null"),
    ("mc_kv_plan", dict(slots=0xc04), "8-byte"),
    ("mc_kv_plan", dict(seq_lens=0x200), "new_lens"),
    ("mc_kv_release", dict(n_req=-1), "n_req"),
    ("mc_kv_release", dict(done=None), "null"),
    ("mc_kv_release", dict(block_size=-16), "block size"),
    ("mc_qk_norm_rope", dict(head_dim=96), "head_dim"),
    ("mc_qk_norm_rope", dict(kv_dtype=_lib.DTYPE_F32), "dtype"),
    ("mc_qk_norm_rope", dict(n_tokens=-1), "n_tokens"),
    ("mc_qk_norm_rope", dict(n_kv_heads=0), "n_kv_heads"),
    ("mc_qk_norm_rope", dict(rot_dim=24), "rot_dim"),
    ("mc_qk_norm_rope", dict(rot_dim=80), "rot_dim"),
    ("mc_qk_norm_rope", dict(positions=None), "null"),
    ("mc_qk_norm_rope", dict(k=None), "null"),
    ("mc_qk_norm_rope", dict(q=0x1000008), "16-byte"),
    ("mc_qk_norm_rope", dict(v=0x3000002), "16-byte"),
    ("mc_qk_norm_rope", dict(k_stride=516), "strides"),
    ("mc_qk_norm_rope", dict(q_out_stride=1024), "overlap"),
    ("mc_qk_norm_rope", dict(q_out=0x1000010), "overlaps q"),
    ("mc_qk_norm_rope", dict(q_out=0x2000000), "overlaps k or v"),
    ("mc_qk_norm_rope", dict(eps=INF), "eps"),
    ("mc_qk_norm_rope", dict(k=0x100000), "in the cache"),
    ("mc_qk_norm_rope", dict(v=0x200400), "in the cache"),
    ("mc_qk_norm_rope", dict(n_tokens=(1 << 30) + 1), "n_tokens"),
    ("mc_qk_norm_rope", dict(block_stride=8 * 16 * 64 - 64), "block stride"),
    ("mc_qk_norm_rope", dict(block_stride=8 * 16 * 64 + 8), "multiple of head_dim"),
    ("mc_qk_norm_rope", dict(k_cache=0x100008), "16-byte"),
    ("mc_qk_norm_rope", dict(k_scale=0x100), "e4m3"),
    ("mc_paged_attention", dict(n_rows=-1), "n_rows"),
    ("mc_paged_attention", dict(n_heads=30), "query heads"),
    ("mc_paged_attention", dict(head_dim=256), "head_dim"),
    ("mc_paged_attention", dict(n_req=3), "row_req"),
    ("mc_paged_attention", dict(table_width=0), "block table"),
    ("mc_paged_attention", dict(window=-1), "window"),
    ("mc_paged_attention", dict(scale=float("nan")), "scale"),
    ("mc_paged_attention", dict(q=0x1000004), "16-byte"),
    ("mc_paged_attention", dict(q_stride=2050), "strides"),
    ("mc_paged_attention", dict(out_stride=64), "overlap"),
    ("mc_paged_attention", dict(out=0x1000000), "overlaps q"),
    ("mc_paged_attention", dict(workspace=None), "null"),
    ("mc_paged_attention", dict(ws_bytes=1000), "workspace"),
    ("mc_paged_attention", dict(workspace=0x3000008), "workspace"),
    ("mc_paged_attention", dict(num_blocks=0), "blocks"),
    ("mc_paged_attention", dict(num_blocks=1 << 25), "2^32"),
    ("mc_logits_process", dict(dtype=_lib.DTYPE_E4M3), "dtype"),
    ("mc_logits_process", dict(vocab=0), "vocab"),
    ("mc_logits_process", dict(batch=65536), "batch"),
    ("mc_logits_process", dict(repetition=None), "seen and repetition"),
    ("mc_logits_process", dict(counts=None), "counts"),
    ("mc_logits_process", dict(frequency=None, presence=None), "counts"),
    ("mc_logits_process", dict(bias_ids=None), "bias"),
    ("mc_logits_process", dict(n_bias=-1), "bias"),
    ("mc_logits_process", dict(n_allowed=1), "mask rows"),
    ("mc_logits_process", dict(allowed=None, allowed_row=0x100), "allowed_row"),
    ("mc_logits_process", dict(logits=0x1000001), "misaligned"),
    ("mc_logits_process", dict(keys=0xa04), "misaligned"),
    ("mc_logits_process", dict(out=0x1000002), "overlaps"),
    ("mc_logits_process", dict(out_stride=500), "overlap"),
    ("mc_logits_mark", dict(seen=None, counts=None), "null"),
    ("mc_logits_mark", dict(batch=-1), "batch"),
    # rows of one stride interleave (parts of a fused row) but share no byte
    ("mc_qk_norm_rope", dict(q_out=0x1000000, k=0x1000010, k_stride=2048), "overlaps k or v"),
    ("mc_qk_norm_rope", dict(q_out=0x1000000, q_stride=2560, q_out_stride=2560, v=0x1001400 - 16, v_stride=2560),
     "overlaps k or v"),
    ("mc_qk_norm_rope", dict(n_tokens=1, q_out=0x2000000 - 4096 + 16, q_out_stride=1 << 20), "overlaps k or v"),
    ("mc_qk_norm_rope", dict(q_out=0x4000000, q=0x4001000, q_stride=2040), "overlaps q"),
    ("mc_qk_norm_rope", dict(q=0x100000), "in the cache"),
    ("mc_qk_norm_rope", dict(q_out=0x200400), "in the cache"),
    # a stride whose product with the pages passes 64 bits
    ("mc_qk_norm_rope", dict(num_blocks=257, block_stride=1 << 62), "2^32"),
    ("mc_paged_attention", dict(num_blocks=257, block_stride=1 << 62), "2^32"),
    ("mc_logits_mark", dict(seen=0x202), "misaligned"),
    ("mc_logits_mark", dict(counts=0x301), "misaligned"),
]


@pytest.mark.parametrize("name,changed,words", REFUSED, ids=[f"{n}-{'-'.join(c)}-{i}" for i, (n, c, _) in enumerate(REFUSED)])
def test_refusals(lib, name, changed, words):
    rc, why = answer(lib, name, **changed)
    assert rc in (_lib.MC_EINVAL, _lib.MC_EUNSUPPORTED) and words in why, why


@pytest.mark.parametrize("name,changed", [
    ("mc_qk_norm_rope", dict(q_out=0x1000000, q_out_stride=2048)),          # in place
    ("mc_qk_norm_rope", dict(v=None, q_norm_w=None, k_norm_w=None, slots=None)),
    ("mc_qk_norm_rope", dict(rot_dim=0, positions=None, turns=None)),
    ("mc_qk_norm_rope", dict(kv_dtype=_lib.DTYPE_E4M3, k_scale=0x600, v_scale=0x700)),
    ("mc_qk_norm_rope", dict(num_blocks=1, block_size=1, block_stride=0)),
    ("mc_qk_norm_rope", dict(num_blocks=1, block_stride=1 << 62)),           # one page: no distance
    ("mc_qk_norm_rope", dict(n_kv_heads=4, q_stride=2560, k=0x1001000, k_stride=2560, v=0x1001200, v_stride=2560,
                             q_out=0x1000000, q_out_stride=2560)),           # in place in a fused row
    ("mc_qk_norm_rope", dict(q_stride=4608, q_out=0x1001000, q_out_stride=4608)),  # beside q in its rows
    ("mc_paged_attention", dict(row_req=0x500, n_rows=1000)),
    ("mc_paged_attention", dict(n_heads=8)),
    ("mc_logits_process", dict(out=0x1000000)),                              # in place
    ("mc_logits_process", dict(seen=None, repetition=None, counts=None, frequency=None, presence=None, keys=None)),
    ("mc_logits_process", dict(allowed_row=0x100, n_allowed=1)),
    ("mc_logits_process", dict(bias_ids=None, bias_vals=None, n_bias=0)),
    ("mc_logits_mark", dict(counts=None)),
])
def test_allowed_variants_reach_the_context(lib, name, changed):
    rc, why = answer(lib, name, **changed)
    assert rc == _lib.MC_EINVAL and "null context" in why, why


@pytest.mark.parametrize("name,changed", [("mc_qk_norm_rope", dict(n_tokens=0, q=None, k=None, v=None, q_out=None)),
                                          ("mc_paged_attention", dict(n_rows=0, q=None, out=None, kv_lens=None)),
                                          ("mc_logits_process", dict(batch=0, logits=None, out=None)),
                                          ("mc_logits_mark", dict(batch=0, tokens=None))])
def test_nothing_to_do_is_no_error(lib, name, changed):
    rc, why = answer(lib, name, **changed)
    assert rc == 0, why


@pytest.mark.parametrize("rot,theta,scale", [(64, 1e6, 1.0), (128, 1e4, 0.25), (16, 5e5, 8.0), (2, 2.0, 1.0)])
def test_rope_turns_are_the_frequencies(lib, rot, theta, scale):
    from fractions import Fraction

    from molten_b200 import kv
    t = kv.rope_turns(rot, theta, scale)
    assert t.dtype == torch.int64 and t.shape == (rot // 2,)
    for i, v in enumerate(t.tolist()):
        f = scale * theta ** (-2 * i / rot) / (2 * math.pi)
        off = Fraction(v % 2 ** 64, 2 ** 64) - Fraction(f)
        off -= round(off)  # whole turns do not matter
        # pow, the product and the quotient round in 53 bits each, 2 pi in the divisor too
        assert abs(off) <= 5 * 2.0 ** -53 * max(f, 2.0 ** -11), (i, float(off))


@pytest.mark.parametrize("args,words", [((0.0, 1.0, 64), "theta"), ((INF, 1.0, 64), "theta"), ((1e6, -1.0, 64), "position_scale"),
                                        ((1e6, 1.0, 63), "rot_dim"), ((1e6, 1.0, 0), "rot_dim")])
def test_rope_turns_refusals(lib, args, words):
    out = (C.c_uint64 * 64)()
    assert lib.mc_rope_turns(*args, out) == _lib.MC_EINVAL
    assert words in lib.mc_last_error().decode()


def test_workspace_sizes(lib):
    assert lib.mc_paged_attention_workspace_bytes(96) == 0
    assert 0 < lib.mc_paged_attention_workspace_bytes(64) < lib.mc_paged_attention_workspace_bytes(128) < 1 << 26


def test_python_checks_come_first():
    from molten_b200 import kv, sample

    class Ctx:
        device, index = torch.device("cuda", 0), 0
        handle = property(lambda s: pytest.fail("the call went on"))

    ctx = Ctx()
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="alike"):
        kv.KvCache(bf(2, 1, 4, 64), bf(2, 1, 4, 128))
    with pytest.raises(ValueError, match="BF16"):
        kv.KvCache(torch.zeros(2, 1, 4, 64), torch.zeros(2, 1, 4, 64))
    with pytest.raises(ValueError, match="contiguous"):
        kv.KvCache(bf(2, 4, 2, 64).transpose(1, 2), bf(2, 4, 2, 64).transpose(1, 2))
    with pytest.raises(ValueError, match="scales"):
        kv.KvCache(bf(2, 2, 4, 64), bf(2, 2, 4, 64), k_scale=torch.zeros(3))
    both = bf(5, 2, 2, 4, 64)
    halves = kv.KvCache(both[:, 0], both[:, 1])
    assert halves._where[2:] == (_lib.DTYPE_BF16, 5, 4, 2 * 2 * 4 * 64)
    with pytest.raises(ValueError, match="empty"):
        kv.KvCache(bf(0, 1, 4, 64), bf(0, 1, 4, 64))
    with pytest.raises(AttributeError):
        halves.k = bf(5, 2, 4, 64)  # its address is taken
    with pytest.raises(ValueError, match="rot_dim"):
        kv.rope_turns(-2)
    one = torch.zeros(3, 128, dtype=torch.bfloat16).as_strided((1, 2, 64), (101, 64, 1))
    here = type("Here", (), dict(device=torch.device("cpu"), index=-1))()
    assert kv._rows(here, one, one.shape, "q") == (one.data_ptr(), 128)  # a single row's stride says nothing
    with pytest.raises(ValueError, match="query heads"):
        kv.paged_attention(ctx, bf(1, 3, 64), halves, i32(1, 5), i32(1), bf(1, 3, 64), i32(4))
    with pytest.raises(ValueError, match="must be on"):
        kv.paged_attention(ctx, bf(1, 4, 64), halves, i32(1, 5), i32(1), bf(1, 4, 64), i32(4))
    with pytest.raises(ValueError, match="k rows"):
        kv.qk_norm_rope(ctx, bf(1, 4, 64), bf(1, 1, 64), None, None, None, None, None, bf(1, 4, 64), halves)
    with pytest.raises(ValueError, match="block table"):
        kv.kv_plan(ctx, i32(3), None, 4, i32(2, 5), i32(9), i32(1), i32(3), i32(1), i32(4), i32(3), i32(3), i32(3),
                   torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="BF16 or F32"):
        sample.logits_process(ctx, torch.zeros(1, 8).half(), torch.zeros(1, 8).half(), sample.LogitsRules())


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_split_of_the_attention_work(tmp_path):
    exe = tmp_path / "split"
    r = subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", str(ROOT / "tests" / "cpp" / "test_paged_split.cpp"),
                        "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok (0 failures)", r.stdout


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_cpp_host_mirror_of_the_serving_calls(lib, tmp_path):
    so = build.build()
    exe = tmp_path / "serving"
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", str(ROOT / "include"),
                        str(ROOT / "tests" / "cpp" / "test_host_mirror_serving.cpp"), "-L", str(so.parent), "-lmolten_cuda",
                        f"-Wl,-rpath,{so.parent}", "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok (0 failures)", r.stdout
