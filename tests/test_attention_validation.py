"""Refusals of the attention operators: the C entry points' status codes and the Python checks that need no GPU, the
argument structs' layout, and the rotary frequency tables."""
from __future__ import annotations

import ctypes
import math
import pathlib
import shutil
import subprocess

import pytest
import torch

ROOT = pathlib.Path(__file__).resolve().parent.parent
PTR = 1 << 20  # a nonzero, aligned address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    from svdflash_b200 import _build, _lib
    if _build.is_stale():
        _build.build()
    return _lib.load()


def _structs():
    from svdflash_b200 import _lib
    return {"rope": (_lib.RopeArgs, _lib.ROPE_ARGS), "pages": (_lib.PagesArgs, _lib.PAGES_ARGS),
            "prompt": (_lib.PromptArgs, _lib.PROMPT_ARGS), "tree": (_lib.TreeArgs, _lib.TREE_ARGS)}


GOOD = {
    "rope": dict(dtype=0, tokens=4, q_heads=8, kv_heads=2, head_dim=128, rotary_dim=128, block_size=16, num_blocks=9,
                 scale=1.0, q=PTR, k=PTR, v=PTR, positions=PTR, slots=PTR, inv_freq=PTR, q_out=PTR, k_out=PTR,
                 k_cache=PTR, v_cache=PTR, k_block=2 * 16 * 128, v_block=2 * 16 * 128, q_token=1024, q_head=128,
                 k_token=256, k_head=128, v_token=256, v_head=128),
    "pages": dict(batch=4, tokens=9, block_size=16, table_width=5, free_capacity=7, table=PTR, ld_table=5, held=PTR,
                  added=PTR, free_blocks=PTR, free_count=PTR, slots=PTR, positions=PTR, cu=PTR, lens=PTR, count_out=PTR,
                  missing=PTR),
    "prompt": dict(dtype=0, batch=2, q_tokens=9, k_tokens=9, q_heads=8, kv_heads=2, head_dim=128, causal=1, scale=0.1,
                   q=PTR, k=PTR, v=PTR, q_token=1024, q_head=128, k_token=256, k_head=128, v_token=256, v_head=128,
                   cu_q=PTR, cu_k=PTR, out=PTR, out_token=1024, out_head=128, workspace=PTR, workspace_bytes=1 << 30),
    "tree": dict(dtype=0, batch=2, tokens=9, q_heads=8, kv_heads=2, head_dim=128, block_size=16, num_blocks=9,
                 table_width=5, max_tree=8, scale=0.1, q=PTR, q_token=1024, q_head=128, k_cache=PTR, v_cache=PTR,
                 k_block=2 * 16 * 128, v_block=2 * 16 * 128, table=PTR, ld_table=5, lens=PTR, cu_q=PTR, out=PTR,
                 out_token=1024, out_head=128, workspace=PTR, workspace_bytes=1 << 30),
}
INVALID, SHAPE, ALIGN, DTYPE, WORKSPACE = -1, -2, -3, -4, -5
BAD = [
    ("rope", dict(q=0), INVALID), ("rope", dict(positions=0), INVALID), ("rope", dict(inv_freq=0), INVALID),
    ("rope", dict(q_out=0), INVALID), ("rope", dict(tokens=0), INVALID), ("rope", dict(q_heads=-1), INVALID),
    ("rope", dict(dtype=2), DTYPE), ("rope", dict(rotary_dim=0), SHAPE), ("rope", dict(rotary_dim=63), SHAPE),
    ("rope", dict(rotary_dim=130), SHAPE), ("rope", dict(head_dim=1024, rotary_dim=64), SHAPE),
    ("rope", dict(scale=math.nan), INVALID), ("rope", dict(v_cache=0), INVALID), ("rope", dict(v=0), INVALID),
    ("rope", dict(slots=0), INVALID), ("rope", dict(block_size=0), INVALID), ("rope", dict(num_blocks=0), INVALID),
    ("rope", dict(k_block=4095), SHAPE), ("rope", dict(k_cache=0, v_cache=0, k_out=0), INVALID),
    ("rope", dict(q=PTR + 1), ALIGN),
    ("pages", dict(table=0), INVALID), ("pages", dict(batch=0), INVALID), ("pages", dict(tokens=-1), INVALID),
    ("pages", dict(block_size=0), INVALID), ("pages", dict(ld_table=4), SHAPE), ("pages", dict(slots=0), INVALID),
    ("pages", dict(free_blocks=0), INVALID), ("pages", dict(missing=0), INVALID),
    ("prompt", dict(k=0), INVALID), ("prompt", dict(cu_k=0), INVALID), ("prompt", dict(batch=0), INVALID),
    ("prompt", dict(k_tokens=0), INVALID), ("prompt", dict(dtype=-1), DTYPE), ("prompt", dict(q_heads=9), SHAPE),
    ("prompt", dict(head_dim=96), SHAPE), ("prompt", dict(scale=math.inf), INVALID), ("prompt", dict(q=PTR + 8), ALIGN),
    ("prompt", dict(v_token=260), ALIGN), ("prompt", dict(out_head=132), ALIGN), ("prompt", dict(workspace=0), INVALID),
    ("prompt", dict(workspace=PTR + 16), INVALID), ("prompt", dict(workspace_bytes=16), WORKSPACE),
    ("tree", dict(lens=0), INVALID), ("tree", dict(max_tree=0), INVALID), ("tree", dict(tokens=0), INVALID),
    ("tree", dict(dtype=7), DTYPE), ("tree", dict(kv_heads=3), SHAPE), ("tree", dict(head_dim=32), SHAPE),
    ("tree", dict(block_size=24), SHAPE), ("tree", dict(block_size=4), SHAPE), ("tree", dict(v_block=4088), SHAPE),
    ("tree", dict(ld_table=4), SHAPE), ("tree", dict(k_cache=PTR + 2), ALIGN), ("tree", dict(k_block=4100), ALIGN),
    ("tree", dict(workspace_bytes=255), WORKSPACE), ("tree", dict(scale=math.nan), INVALID),
]
ENTRY = {"rope": "svdmlp_rope", "pages": "svdmlp_page_step", "prompt": "svdmlp_prompt_attention",
         "tree": "svdmlp_tree_attention"}


@pytest.mark.parametrize("op,change,status", BAD)
def test_entry_points_refuse(lib, op, change, status):
    mirror, _ = _structs()[op]
    args = mirror(**{**GOOD[op], **change})
    assert getattr(lib, ENTRY[op])(ctypes.addressof(args), None) == status


@pytest.mark.parametrize("op", sorted(ENTRY))
def test_entry_points_refuse_null_arguments(lib, op):
    assert getattr(lib, ENTRY[op])(None, None) == INVALID


def test_workspace_sizes(lib):
    assert lib.svdmlp_prompt_workspace_bytes() >= 256
    assert lib.svdmlp_tree_workspace_bytes(128) >= 256
    assert lib.svdmlp_tree_workspace_bytes(96) == SHAPE


def test_packed_arguments_lie_as_the_mirror_says():
    for name, (mirror, pack) in _structs().items():
        values = [i + 1 for i in range(len(mirror._fields_))]
        raw = pack(*values)
        assert len(raw) == ctypes.sizeof(mirror), name
        got = mirror.from_buffer_copy(raw)
        assert [getattr(got, f) for f, _ in mirror._fields_] == values, name


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_structs_match_the_header(tmp_path):
    """Every field's offset, as a C compiler sees include/svdmlp.h."""
    lines, want = [], []
    for name, (mirror, _) in _structs().items():
        for f, _kind in mirror._fields_:
            lines.append(f'printf("%zu\\n", offsetof(svdmlp_{name}_args, {f}));')
            want.append(getattr(mirror, f).offset)
        lines.append(f'printf("%zu\\n", sizeof(svdmlp_{name}_args));')
        want.append(ctypes.sizeof(mirror))
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "svdmlp.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == want


def test_python_refuses_what_is_not_on_the_gpu():
    from svdflash_b200.kernels import attention as att
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    cu = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        att.prompt_attention(x, x, x, cu)
    with pytest.raises(ValueError, match="CUDA"):
        att.rope(x, x, cu, torch.ones(32))
    with pytest.raises(TypeError, match="torch.Tensor"):
        att.prompt_attention([1], x, x, cu)
    with pytest.raises(ValueError, match="CUDA"):
        att.page_step(torch.zeros(1, 2, dtype=torch.int32), cu, cu, cu, cu, 16, 1)
    with pytest.raises(TypeError, match="int32"):
        att.page_step(torch.zeros(1, 2), cu, cu, cu, cu, 16, 1)
    with pytest.raises(ValueError, match="positive integer"):
        att.kv_cache(0, 1, 16, 64, device="cpu")


@pytest.mark.parametrize("bad", [dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=130), dict(base=0.0),
                                 dict(scaling=dict(type="spiral")),
                                 dict(scaling=dict(rope_type="llama3", factor=8, low_freq_factor=4, high_freq_factor=4,
                                                   original_max_position_embeddings=8192))])
def test_rope_frequencies_refuse(bad):
    from svdflash_b200.kernels import attention as att
    with pytest.raises(ValueError):
        att.rope_frequencies(128, device="cpu", **bad)


def test_rope_frequencies():
    from svdflash_b200.kernels import attention as att
    d, base = 128, 500000.0
    plain, one = att.rope_frequencies(d, base=base, device="cpu")
    want = base ** (-torch.arange(64, dtype=torch.float64) / 64)
    assert one == 1.0 and torch.equal(plain, want.float())
    part, _ = att.rope_frequencies(d, base=base, rotary_dim=32, device="cpu")
    assert torch.equal(part, (base ** (-torch.arange(16, dtype=torch.float64) / 16)).float())
    lin, one = att.rope_frequencies(d, base=base, scaling=dict(type="linear", factor=4.0), device="cpu")
    assert one == 1.0 and torch.equal(lin, (want / 4).float())
    # llama3: short waves kept, long ones divided, a blend between that decreases all the way
    s = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
             original_max_position_embeddings=8192)
    got = att.rope_frequencies(d, base=base, scaling=s, device="cpu")[0].double()
    wave = 2 * math.pi / want
    assert torch.allclose(got[wave < 8192 / 4], want[wave < 8192 / 4], rtol=1e-6)
    assert torch.allclose(got[wave > 8192], want[wave > 8192] / 8, rtol=1e-6)
    mid = (wave >= 8192 / 4) & (wave <= 8192)
    blend = (8192 / wave[mid] - 1.0) / 3.0
    assert mid.any() and torch.allclose(got[mid], (1 - blend) * want[mid] / 8 + blend * want[mid], rtol=1e-6)
    assert (got[1:] < got[:-1]).all()
    # yarn: the ends as above, and the magnitude
    y, magnitude = att.rope_frequencies(d, base=10000.0, scaling=dict(
        type="yarn", factor=16.0, original_max_position_embeddings=4096), device="cpu")
    base_freq = 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    turns = 4096 * base_freq / (2 * math.pi)
    assert magnitude == pytest.approx(0.1 * math.log(16.0) + 1.0)
    assert torch.allclose(y.double()[turns > 34], base_freq[turns > 34], rtol=1e-6)
    assert torch.allclose(y.double()[turns < 0.9], base_freq[turns < 0.9] / 16, rtol=1e-6)
    assert att.rope_frequencies(d, scaling=dict(type="yarn", factor=4.0, original_max_position_embeddings=4096,
                                                attention_factor=1.5), device="cpu")[1] == 1.5
