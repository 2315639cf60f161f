"""The decoder's calibration pass follows the attention that the decoder runs: per-head norms, window and first tokens.

The largest output of the first layer's attention in each channel, against plain fp32 attention on the same bf16 queries, keys and
values.  Bound: the kernel rounds the weights and the output to bf16, 3 x 2^-8 of the largest |v|, and a query or key may round the
other way after fp32 norms and rotations in another order, 2^-8 more at most.
"""

import pytest
import torch
import torch.nn.functional as F

from fms_model_optimizer_b200.decoder import W8A8Decoder, calibrate_act_scales, linear_shapes, synth_weight

pytestmark = pytest.mark.gpu

CFG = dict(layers=1, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, ffn=2048, vocab=2048, rope_theta=10000.0, batch=2, seq=96)


def _plain_attention_max(cfg, dev, ids):
    """(largest |output| of every channel behind the first layer's attention, largest |v|), from the model's own weights and norms."""
    model = W8A8Decoder(cfg, dev, layers=1)
    B, S = ids.shape
    hd, nkv = cfg["head_dim"], cfg["kv_heads"]
    group = cfg["q_heads"] // nkv
    w = {name: synth_weight(n, k, ni, dev) for ni, (name, (n, k, _)) in enumerate(linear_shapes(cfg).items()) if name in "qkv"}
    h = F.rms_norm(F.embedding(ids, model.embed).view(B * S, -1), (cfg["hidden"],), model.layers[0]["ln1"], 1e-5)
    c, s = (t[:S, None].repeat(B, 1, 1) for t in (model.cos, model.sin))

    def heads(name, norm):
        x = F.linear(h, w[name]).view(B * S, -1, hd).float()
        if norm is not None:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * norm.float()
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1).bfloat16().float().view(B, S, -1, hd)

    q, k = heads("q", model.layers[0]["q_norm"]), heads("k", model.layers[0]["k_norm"])
    v = F.linear(h, w["v"]).view(B, S, nkv, hd).float()
    x = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(group, 2)) * hd**-0.5
    i, j = torch.arange(S, device=dev)[:, None], torch.arange(S, device=dev)[None]
    seen = j <= i
    if cfg.get("window", 0):
        seen &= (j > i - cfg["window"]) | (j < cfg.get("sinks", 0))
    out = torch.einsum("bhij,bjhd->bihd", x.masked_fill(~seen, -torch.inf).softmax(-1), v.repeat_interleave(group, 2))
    return out.reshape(B * S, -1).abs().amax(0), float(v.abs().max())


@pytest.mark.parametrize("extra", [{}, dict(qk_norm=True), dict(window=3, sinks=1), dict(qk_norm=True, window=20)])
def test_calibration_runs_the_decoders_attention(cuda_dev, extra):
    cfg = dict(CFG, **extra)
    ids = torch.randint(0, cfg["vocab"], (2, 96), generator=torch.Generator().manual_seed(3)).to(cuda_dev)
    got = calibrate_act_scales(cfg, cuda_dev, ids, 1)
    want, most = _plain_attention_max(cfg, cuda_dev, ids)
    assert float((got[(0, "o")] - want).abs().max()) <= 4 * 2.0**-8 * most
    assert set(got) == {(0, name) for name in linear_shapes(cfg)}
