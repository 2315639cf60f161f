"""CPU checks of the C interface of the operators that answer many requests at once: argument blocks, refusals, and that there is no CPU path."""

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
STRUCTS = (("qlin_token_logprobs_args", L.TokenLogprobsArgs), ("qlin_lora_args", L.LoraArgs), ("qlin_prefix_attention_args", L.PrefixAttentionArgs))


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


def test_refusals_of_the_token_log_probabilities():
    lib = L.load()
    buf, base = _base()
    good = dict(logits=base, tokens=base, logprobs=base, entropy=base, stats=base, top_logprobs=base, top_ids=base, d_logits=base, ld=64, rows=1, vocab=64, top=3, dtype=L.DT_BF16)

    for fn in (lib.qlin_token_logprobs, lib.qlin_token_logprobs_bwd):

        def rc(**kw):
            return fn(C.byref(L.TokenLogprobsArgs(**{**good, **kw})), None)

        assert fn(None, None) == L.ERR_NULL and rc(rows=0) == L.OK
        assert rc(logits=None) == L.ERR_NULL and rc(tokens=None) == L.ERR_NULL and rc(entropy=None) == L.ERR_NULL
        assert rc(rows=-1) == L.ERR_BAD_SHAPE and rc(vocab=0) == L.ERR_BAD_SHAPE and rc(top=-1) == L.ERR_BAD_SHAPE and rc(ld=-1) == L.ERR_BAD_SHAPE
        assert rc(top=33) == L.ERR_BAD_SHAPE and rc(vocab=2) == L.ERR_BAD_SHAPE and rc(vocab=(1 << 20) + 1) == L.ERR_TOO_LARGE
        assert rc(dtype=L.DT_I8) == L.ERR_BAD_DTYPE and rc(logits=base + 1) == L.ERR_BAD_ALIGN and rc(dtype=L.DT_F32, logits=base + 2) == L.ERR_BAD_ALIGN
    assert lib.qlin_token_logprobs(C.byref(L.TokenLogprobsArgs(**{**good, "top_ids": None})), None) == L.ERR_NULL
    assert lib.qlin_token_logprobs_bwd(C.byref(L.TokenLogprobsArgs(**{**good, "stats": None})), None) == L.ERR_NULL
    assert lib.qlin_token_logprobs_bwd(C.byref(L.TokenLogprobsArgs(**{**good, "d_logits": base + 1})), None) == L.ERR_BAD_ALIGN


def test_refusals_of_the_adapters():
    lib = L.load()
    buf, base = _base()
    good = dict(x=base, a=base, b=base, y=base, rows=base, starts=base, scale=base, x_row=64, y_row=64, a_adapter=1024, a_row=64, b_adapter=1024, b_row=16, tokens=1, listed=1,
                adapters=1, rank=16, width=64, out=64, dtype=L.DT_BF16)  # fmt: skip

    def rc(**kw):
        return lib.qlin_lora(C.byref(L.LoraArgs(**{**good, **kw})), None)

    assert lib.qlin_lora(None, None) == L.ERR_NULL
    assert rc(listed=0) == L.OK and rc(adapters=0) == L.OK and rc(out=0) == L.OK and rc(width=0) == L.OK
    assert rc(x=None) == L.ERR_NULL and rc(starts=None) == L.ERR_NULL and rc(scale=None) == L.ERR_NULL
    assert rc(tokens=-1) == L.ERR_BAD_SHAPE and rc(rank=0) == L.ERR_BAD_SHAPE and rc(rank=12) == L.ERR_BAD_SHAPE and rc(rank=136) == L.ERR_BAD_SHAPE
    assert rc(width=60) == L.ERR_BAD_SHAPE and rc(out=4) == L.ERR_BAD_SHAPE and rc(listed=(1 << 27) + 1) == L.ERR_TOO_LARGE
    assert rc(dtype=L.DT_F32) == L.ERR_BAD_DTYPE and rc(y=base + 8) == L.ERR_BAD_ALIGN and rc(b_row=20) == L.ERR_BAD_ALIGN


def test_refusals_of_the_attention_behind_a_prefix():
    lib = L.load()
    buf, base = _base()
    own = dict(q=base, k_pages=base, v_pages=base, block_table=base, lens=base, out=base, workspace=base, q_batch=64, q_head=64, page_stride=64, head_stride=64,
               slot_stride=64, table_stride=1, batch=1, q_heads=2, kv_heads=1, head_dim=64, page_size=1, num_pages=1, max_pages=1, dtype=L.DT_BF16,
               cache_dtype=L.DT_BF16, scale=0.125)  # fmt: skip
    good = dict(prefix_table=base, prefix_lens=base, groups=base, prefix_stride=1, num_groups=1, max_prefix_pages=1)

    def rc(kw={}, **own_kw):
        return lib.qlin_prefix_attention(C.byref(L.PrefixAttentionArgs(own=L.PagedAttentionArgs(**{**own, **own_kw}), **{**good, **kw})), None)

    assert lib.qlin_prefix_attention(None, None) == L.ERR_NULL and rc(batch=0) == L.OK
    assert rc(q=None) == L.ERR_NULL and rc(dict(groups=None)) == L.ERR_NULL and rc(dict(prefix_table=None)) == L.ERR_NULL and rc(workspace=None) == L.ERR_NULL
    assert rc(dict(num_groups=0)) == L.ERR_BAD_SHAPE and rc(dict(max_prefix_pages=-1)) == L.ERR_BAD_SHAPE and rc(dict(num_groups=(1 << 20) + 1)) == L.ERR_TOO_LARGE
    assert rc(dict(max_prefix_pages=1 << 20), page_size=1 << 11) == L.ERR_TOO_LARGE
    assert rc(q_heads=3, kv_heads=2) == L.ERR_BAD_SHAPE and rc(head_dim=60) == L.ERR_BAD_SHAPE and rc(dtype=L.DT_F32) == L.ERR_BAD_DTYPE
    assert rc(k_pages=base + 8) == L.ERR_BAD_ALIGN and rc(workspace=base + 4) == L.ERR_BAD_ALIGN
    a = L.PrefixAttentionArgs(own=L.PagedAttentionArgs(**{**own, "head_dim": 60}), **good)
    assert lib.qlin_prefix_attention_workspace_bytes(C.byref(a)) == L.ERR_BAD_SHAPE


def test_no_cpu_path():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.token_logprobs(x, torch.zeros(2, dtype=torch.long))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.lora_add_(x, x, x[None, :1], x[None, :, :1], *ops.lora_groups(torch.zeros(2, dtype=torch.long), 1), torch.ones(1))


def test_the_rows_of_each_adapter():
    which = torch.tensor([2, -1, 0, 2, 7, 1, 0, -100, 2])
    rows, starts = ops.lora_groups(which, 4)
    assert starts.tolist() == [0, 2, 3, 6, 6] and rows[:6].tolist() == [2, 6, 5, 0, 3, 8]
