"""What the attention calls promise around their arithmetic: gradients refused, outputs that overlap inputs, caches without room."""

import ctypes as C
import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from fms_model_optimizer_b200 import _lib as L
from fms_model_optimizer_b200 import ops

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g).to(dtype)


class _Calls:
    """The three calls with every floating-point argument by name."""

    def __init__(self, dev, f8):
        g = torch.Generator().manual_seed(31)
        r = lambda *shape, dtype=torch.bfloat16: _randn(g, *shape, dtype=dtype).to(dev)  # noqa: E731
        self.i = torch.tensor([0, 1], dtype=torch.int32, device=dev)
        self.cu = torch.tensor([0, 2], dtype=torch.int32, device=dev)
        self.n = torch.tensor([3, 7], dtype=torch.int32, device=dev)
        pages = lambda: r(4, 2, 8, 64, dtype=torch.float32).to(F8 if f8 else torch.bfloat16)  # noqa: E731
        scales = dict(k_scale=torch.ones(2, device=dev), v_scale=torch.ones(2, device=dev)) if f8 else {}
        qkv = dict(q=r(2, 4, 64), k=r(2, 2, 64), v=r(2, 2, 64))
        self.args = {
            "rotate": dict(qkv, cos=r(4, 32, dtype=torch.float32), sin=r(4, 32, dtype=torch.float32), q_weight=r(64), k_weight=r(64), k_pages=pages(), v_pages=pages(), **scales),
            "token": dict(q=r(2, 4, 64), k_pages=pages(), v_pages=pages(), out=r(2, 4, 64), **scales),
            "prompt": dict(qkv, out=r(2, 4, 64)),
        }

    def __call__(self, which, **other):
        a = dict(self.args[which], **other)
        if which == "rotate":
            return ops.qk_norm_rope(a.pop("q"), a.pop("k"), a.pop("cos"), a.pop("sin"), self.i, slots=self.i.long(), **a)
        if which == "token":
            return ops.paged_attention(a.pop("q"), a.pop("k_pages"), a.pop("v_pages"), self.i[:, None], self.n, **a)
        return ops.prompt_attention(a.pop("q"), a.pop("k"), a.pop("v"), self.cu, self.cu, 2, **a)


@pytest.mark.parametrize("which", ["rotate", "token", "prompt"])
@pytest.mark.parametrize("f8", [False, True])
def test_no_gradient_is_cut_off_silently(cuda_dev, which, f8):
    calls = _Calls(cuda_dev, f8)
    calls(which)
    for name, t in calls.args[which].items():
        if t.dtype != F8:  # no gradient reaches codes
            wanting = t.clone().requires_grad_()
            with pytest.raises(RuntimeError, match="no gradient"):
                calls(which, **{name: wanting})
            with torch.no_grad():
                calls(which, **{name: wanting})
            with fwAD.dual_level(), torch.no_grad():  # tangents pass through no_grad
                dual = fwAD.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match="no gradient"):
                    calls(which, **{name: dual})
    ops.check_status(cuda_dev)
