"""CPU checks of the C interface of the generating decoder's attention: argument blocks, refusals, and that there is no CPU path."""

import ctypes as C
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from fms_model_optimizer_b200 import _lib as L
from fms_model_optimizer_b200 import ops

HEADER = Path(__file__).resolve().parent.parent / "include" / "qlin_b200.h"
STRUCTS = (("qlin_qk_rope_args", L.QkRopeArgs), ("qlin_paged_attention_args", L.PagedAttentionArgs), ("qlin_prompt_attention_args", L.PromptAttentionArgs))


@pytest.mark.parametrize("name,cls", STRUCTS)
def test_argument_block_matches_the_header(tmp_path, name, cls):
    gcc = shutil.which("gcc")
    assert gcc, "gcc is part of this build's toolchain"
    body = re.search(r"typedef struct " + name + r" \{(.*?)\} " + name, HEADER.read_text(), flags=re.S).group(1)
    fields = re.findall(r"\*?(\w+)\s*[,;]", re.sub(r"/\*.*?\*/", "", body, flags=re.S))
    assert fields == [f[0] for f in cls._fields_]
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {", f'printf("%zu\\n", sizeof({name}));']
    lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields] + ["return 0; }"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", "-o", str(exe), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def _base():
    buf = (C.c_char * 8192)()
    return buf, (C.addressof(buf) + 15) // 16 * 16


def test_refusals_of_the_rotation():
    lib = L.load()
    buf, base = _base()
    good = dict(q=base, k=base, v=base, q_out=base, cos=base, sin=base, positions=base, k_pages=base, v_pages=base, slots=base, q_token=64, q_head=64, k_token=64,
                k_head=64, v_token=64, v_head=64, page_stride=64, head_stride=64, slot_stride=64, num_slots=1, tokens=1, q_heads=1, kv_heads=1, head_dim=64,
                rotary=64, table_rows=1, page_size=1, dtype=L.DT_BF16, weight_dtype=L.DT_BF16, cache_dtype=L.DT_BF16)  # fmt: skip

    def rc(**kw):
        return lib.qlin_qk_rope(C.byref(L.QkRopeArgs(**{**good, **kw})), None)

    assert lib.qlin_qk_rope(None, None) == L.ERR_NULL
    assert rc(tokens=0) == L.OK
    assert rc(q=None) == L.ERR_NULL and rc(slots=None) == L.ERR_NULL and rc(cache_dtype=L.DT_F8E4M3) == L.ERR_NULL
    assert rc(tokens=-1) == L.ERR_BAD_SHAPE and rc(head_dim=40) == L.ERR_BAD_SHAPE and rc(head_dim=528) == L.ERR_BAD_SHAPE
    assert rc(rotary=80) == L.ERR_BAD_SHAPE and rc(rotary=8) == L.ERR_BAD_SHAPE and rc(page_size=0) == L.ERR_BAD_SHAPE
    assert rc(dtype=L.DT_I8) == L.ERR_BAD_DTYPE and rc(cache_dtype=L.DT_F32) == L.ERR_BAD_DTYPE
    assert rc(q_weight=base, weight_dtype=L.DT_F16) == L.ERR_BAD_DTYPE
    assert rc(q=base + 2) == L.ERR_BAD_ALIGN and rc(k_head=4) == L.ERR_BAD_ALIGN and rc(slot_stride=20) == L.ERR_BAD_ALIGN


def test_refusals_of_the_attention_over_pages():
    lib = L.load()
    buf, base = _base()
    good = dict(q=base, k_pages=base, v_pages=base, block_table=base, lens=base, out=base, workspace=base, q_batch=64, q_head=64, page_stride=64, head_stride=64,
                slot_stride=64, table_stride=1, batch=1, q_heads=2, kv_heads=1, head_dim=64, page_size=1, num_pages=1, max_pages=1, dtype=L.DT_BF16,
                cache_dtype=L.DT_BF16, scale=0.125)  # fmt: skip

    def rc(**kw):
        a = L.PagedAttentionArgs(**{**good, **kw})
        got = lib.qlin_paged_attention(C.byref(a), None)
        return got

    assert lib.qlin_paged_attention(None, None) == L.ERR_NULL
    assert rc(batch=0) == L.OK
    assert rc(q=None) == L.ERR_NULL and rc(k_pages=None) == L.ERR_NULL and rc(cache_dtype=L.DT_F8E4M3) == L.ERR_NULL
    assert rc(q_heads=3, kv_heads=2) == L.ERR_BAD_SHAPE and rc(head_dim=60) == L.ERR_BAD_SHAPE and rc(head_dim=136) == L.ERR_BAD_SHAPE
    assert rc(head_dim=72, cache_dtype=L.DT_F8E4M3) == L.ERR_BAD_SHAPE and rc(page_size=0) == L.ERR_BAD_SHAPE
    assert rc(dtype=L.DT_F32) == L.ERR_BAD_DTYPE and rc(cache_dtype=L.DT_F16) == L.ERR_BAD_DTYPE
    assert rc(max_pages=1 << 20, page_size=1 << 11) == L.ERR_TOO_LARGE
    assert rc(k_pages=base + 8) == L.ERR_BAD_ALIGN and rc(q_head=20) == L.ERR_BAD_ALIGN
    a = L.PagedAttentionArgs(**{**good, "head_dim": 60})
    assert lib.qlin_paged_attention_workspace_bytes(C.byref(a)) == L.ERR_BAD_SHAPE


def test_refusals_of_the_prompt_attention():
    lib = L.load()
    buf, base = _base()
    good = dict(q=base, k=base, v=base, out=base, cu_q=base, cu_k=base, q_token=64, q_head=64, k_token=64, k_head=64, v_token=64, v_head=64, tokens_q=1, tokens_k=1,
                batch=1, max_q=1, q_heads=2, kv_heads=1, head_dim=64, dtype=L.DT_BF16, scale=0.125)  # fmt: skip

    def rc(**kw):
        return lib.qlin_prompt_attention(C.byref(L.PromptAttentionArgs(**{**good, **kw})), None)

    assert lib.qlin_prompt_attention(None, None) == L.ERR_NULL
    assert rc(tokens_q=0) == L.OK and rc(batch=0) == L.OK
    assert rc(q=None) == L.ERR_NULL and rc(v=None) == L.ERR_NULL and rc(cu_k=None) == L.ERR_NULL
    assert rc(q_heads=3, kv_heads=2) == L.ERR_BAD_SHAPE and rc(head_dim=60) == L.ERR_BAD_SHAPE and rc(head_dim=136) == L.ERR_BAD_SHAPE
    assert rc(q_heads=130) == L.ERR_UNSUPPORTED
    assert rc(dtype=L.DT_F32) == L.ERR_BAD_DTYPE
    assert rc(q=base + 2) == L.ERR_BAD_ALIGN and rc(v_token=4) == L.ERR_BAD_ALIGN


def test_no_cpu_path():
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    t = torch.zeros(1, 32)
    pages = torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.qk_norm_rope(x, x, t, t, i)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attention(x, pages, pages, i[None], i)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.prompt_attention(x, x, x, i, i, 1)
