"""Cases of the serving operators of a decoder's attention: per-head norms of queries and keys with the position rotation
and the write into a paged key-value cache in one pass, attention of whole prompts with a sliding window and first tokens
that stay visible, and attention of one new token over the paged cache.

Query i of a sequence with n queries and m keys stands at position i + m - n and sees the keys at positions
(pos - window, pos] and, whatever the window, the first `sinks` keys (window 0: all keys up to pos).
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
EPS = 1e-6
F8_MAX = 448.0


# ---------------------------------------------------------------------------------------------------- cases
def _rotate(name, tokens, q_heads, kv_heads, head_dim, rotary, dtype, norm, cache, page):
    return dict(name=name, op="qk_norm_rope", tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, rotary=rotary, dtype=dtype, norm=norm,
                cache=cache, page=page)  # fmt: skip


def _token(name, batch, longest, ragged, q_heads, kv_heads, head_dim, dtype, cache, page, window, sinks):
    return dict(name=name, op="paged_attention", batch=batch, longest=longest, ragged=ragged, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype,
                cache=cache, page=page, window=window, sinks=sinks)  # fmt: skip


def _prompt(name, batch, longest, ragged, past, q_heads, kv_heads, head_dim, dtype, window, sinks):
    return dict(name=name, op="prompt_attention", batch=batch, longest=longest, ragged=ragged, past=past, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                dtype=dtype, window=window, sinks=sinks)  # fmt: skip


def listed():
    return [
        # one new token of one sequence: the latency of a layer's step
        _rotate("rotate, 1 token", 1, 32, 8, 128, 128, "bf16", True, "bf16", 16),
        # a decode batch whose cache is held in e4m3
        _rotate("rotate, 64 tokens, e4m3 cache", 64, 32, 8, 128, 128, "bf16", True, "fp8", 64),
        # the prompts of the benchmark's decoder: 8 x 2048 tokens
        _rotate("rotate, 16384 tokens", 16384, 32, 8, 128, 128, "bf16", True, "bf16", 64),
        # an odd number of tokens, small heads of which half is rotated, no norm
        _rotate("rotate, 1999 tokens of 12 x 64", 1999, 12, 12, 64, 32, "fp16", False, "fp16", 24),
        # one sequence of the benchmark's length
        _token("token, 1 x 2048", 1, 2048, False, 32, 8, 128, "bf16", "bf16", 16, 0, 0),
        # a serving batch of ragged lengths, cache in e4m3
        _token("token, 61 x ragged 4099, e4m3", 61, 4099, True, 32, 8, 128, "bf16", "fp8", 64, 0, 0),
        # one long context
        _token("token, 1 x 131072", 1, 131072, False, 32, 8, 128, "bf16", "bf16", 64, 0, 0),
        # long contexts of which a window and the first tokens are visible
        _token("token, 16 x 20001, window 4096", 16, 20001, False, 16, 2, 64, "fp16", "fp16", 48, 4096, 4),
        # the prompts of the benchmark's decoder
        _prompt("prompt, 8 x 2048", 8, 2048, False, 0, 32, 8, 128, "bf16", 0, 0),
        # one long prompt under a window with first tokens that stay visible
        _prompt("prompt, 1 x 8191, window 2048", 1, 8191, False, 0, 32, 8, 128, "bf16", 2048, 4),
        # short ragged prompts that go on after earlier tokens, small heads
        _prompt("prompt, 5 x ragged 333 after 77", 5, 333, True, 77, 12, 12, 64, "fp16", 0, 0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv = rng.choice([(32, 8), (12, 12), (16, 2), (8, 1), (40, 8)])
    dim = rng.choice([64, 96, 128])
    dtype = rng.choice(["bf16", "fp16"])
    page = rng.choice([16, 24, 32, 64, 128])
    op = rng.choice(["qk_norm_rope", "paged_attention", "prompt_attention"])
    if op == "qk_norm_rope":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c = _rotate("", _log(rng, 1, 7000), hq, hkv, dim, rng.choice([dim, dim, dim // 2]), dtype, rng.random() < 0.7, rng.choice([dtype, "fp8", "none"]), page)
    elif op == "paged_attention":
        longest = _log(rng, 1, 80000)
        batch = _log(rng, 1, max(1, min(128, 100000 // longest)))
        window, sinks = rng.choice([(0, 0), (0, 0), (1024, 4), (4096, 1), (129, 0)])
        c = _token("", batch, longest, rng.random() < 0.7, hq, hkv, dim, dtype, rng.choice([dtype, "fp8"]), page, window, sinks)
    else:
        longest, past = _log(rng, 1, 4200), rng.choice([0, 0, _log(rng, 1, 1000)])
        batch = _log(rng, 1, max(1, min(16, 12000000 // (longest * (longest + past)))))
        window, sinks = rng.choice([(0, 0), (0, 0), (1024, 4), (300, 1), (128, 0)])
        c = _prompt("", batch, longest, rng.random() < 0.7, past, hq, hkv, dim, dtype, window, sinks)
    del c["name"]
    return c


def _lengths(case):
    """Lengths of the sequences of a batch; those of a ragged one are spread evenly up to the longest, the longest first."""
    b, n = case["batch"], case["longest"]
    return [max(1, n - (n * i) // b) if case["ragged"] else n for i in range(b)]


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _tables(n, rotary):
    inv = 1.0 / (500000.0 ** (torch.arange(0, rotary, 2, device="cuda").float() / rotary))
    ang = torch.outer(torch.arange(n, device="cuda").float(), inv)
    return ang.cos().contiguous(), ang.sin().contiguous()


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    dt = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "qk_norm_rope":
        t = case["tokens"]
        qkv = _randn(g, (t, (hq + 2 * hkv) * d), dt, 2.0)  # the output of one Linear for q, k and v
        s["q"], s["k"], s["v"] = (x.view(t, -1, d) for x in qkv.split([hq * d, hkv * d, hkv * d], dim=1))
        s["q_weight"] = _randn(g, (d,), dt, 0.1) + 1 if case["norm"] else None
        s["k_weight"] = _randn(g, (d,), dt, 0.1) + 1 if case["norm"] else None
        s["cos"], s["sin"] = _tables(16384 + 64, case["rotary"])
        s["positions"] = torch.randint(0, 64, (1,), generator=g, device="cuda", dtype=torch.int32) + torch.arange(t, device="cuda", dtype=torch.int32)
        s["k_pages"] = s["v_pages"] = s["slots"] = s["k_scale"] = s["v_scale"] = None
        if case["cache"] != "none":
            page = case["page"]
            pages = -(-t // page) + 3
            s["k_pages"], s["v_pages"] = (_randn(g, (pages, hkv, page, d), torch.float32).to(DTYPES[case["cache"]]) for _ in range(2))
            table = torch.randperm(pages, generator=g, device="cuda")
            i = torch.arange(t, device="cuda")
            s["slots"] = table[i // page] * page + i % page
            if case["cache"] == "fp8":
                s["k_scale"], s["v_scale"] = (torch.rand(hkv, generator=g, device="cuda") * 0.03 + 0.01 for _ in range(2))
    elif case["op"] == "paged_attention":
        b, page, longest = case["batch"], case["page"], case["longest"]
        per = -(-longest // page)
        s["q"] = _randn(g, (b, hq, d), dt, 1.5)
        s["k_pages"], s["v_pages"] = (torch.empty((b * per + 1, hkv, page, d), dtype=DTYPES[case["cache"]], device="cuda") for _ in range(2))
        part = max(1, (1 << 27) // (hkv * page * d))
        for pages in (s["k_pages"], s["v_pages"]):  # in parts, so that a long cache needs no fp32 copy of itself
            for i in range(0, pages.shape[0], part):
                pages[i : i + part] = _randn(g, pages[i : i + part].shape, torch.float32).to(pages.dtype)
        s["block_table"] = torch.randperm(b * per, generator=g, device="cuda").to(torch.int32).view(b, per)
        s["lens"] = _int32(_lengths(case))
        s["k_scale"] = s["v_scale"] = None
        if case["cache"] == "fp8":
            s["k_scale"], s["v_scale"] = (torch.rand(hkv, generator=g, device="cuda") * 0.5 + 0.75 for _ in range(2))
    else:
        n = _lengths(case)
        m = [x + case["past"] for x in n]
        s["cu_q"], s["cu_k"] = (_int32([0] + torch.tensor(x).cumsum(0).tolist()) for x in (n, m))
        s["q"] = _randn(g, (sum(n), hq, d), dt, 1.5)
        s["k"], s["v"] = (_randn(g, (sum(m), hkv, d), dt) for _ in range(2))
        s["max_q"], s["max_k"] = max(n), max(m)
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(s):
    if s["op"] == "qk_norm_rope":
        q, k = _own_rotate(s) if own else _plain_rotate(s)
        out = {"q": q, "k": k}
        if s["k_pages"] is not None:
            out.update(k_pages=s["k_pages"], v_pages=s["v_pages"])
        return out
    if s["op"] == "paged_attention":
        return _own_token(s) if own else _plain_token(s)
    return _own_prompt(s) if own else _plain_prompt(s)


def _own_rotate(s):
    from fms_model_optimizer_b200 import ops

    return ops.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS,
                            v=s["v"] if s["k_pages"] is not None else None, k_pages=s["k_pages"], v_pages=s["v_pages"], slots=s["slots"],
                            k_scale=s["k_scale"], v_scale=s["v_scale"])  # fmt: skip


def _own_token(s):
    from fms_model_optimizer_b200 import ops

    return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["lens"], window=s["window"], sinks=s["sinks"], k_scale=s["k_scale"],
                               v_scale=s["v_scale"])  # fmt: skip


def _own_prompt(s):
    from fms_model_optimizer_b200 import ops

    return ops.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["max_q"], window=s["window"], sinks=s["sinks"])


def _plain_heads(x, weight, cos, sin):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half : 2 * half], x[..., 2 * half :]
    c, n = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * n, b * c + a * n, rest], dim=-1)


def _plain_write(pages, slots, values, scale):
    page = pages.shape[2]
    if scale is not None:
        values = (values / scale[:, None]).clamp(-F8_MAX, F8_MAX)
    values = values.to(pages.dtype)
    if pages.dtype == torch.float8_e4m3fn:
        pages, values = pages.view(torch.uint8), values.view(torch.uint8)
    pages[slots // page, :, slots % page] = values


def _plain_rotate(s):
    pos = s["positions"].long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    q, k = _plain_heads(s["q"], s["q_weight"], cos, sin), _plain_heads(s["k"], s["k_weight"], cos, sin)
    if s["k_pages"] is not None:
        _plain_write(s["k_pages"], s["slots"], k, s["k_scale"])
        _plain_write(s["v_pages"], s["slots"], s["v"].float(), s["v_scale"])
    return q.to(s["q"].dtype), k.to(s["k"].dtype)


def _visible(pos, keys, window, sinks):
    seen = keys <= pos
    return seen & ((keys > pos - window) | (keys < sinks)) if window > 0 else seen


def _softmax(scores, seen):
    """Softmax over the visible keys; a row that sees none is zero."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - top.masked_fill(top == -math.inf, 0.0)).exp()
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _gathered(pages, table, scale):
    """[batch, kv heads, keys, head dim] in fp32."""
    x = (pages.view(torch.uint8)[table].view(pages.dtype) if pages.dtype == torch.float8_e4m3fn else pages[table]).float()
    x = x.transpose(1, 2).flatten(2, 3)
    return x if scale is None else x * scale[:, None, None]


def _plain_token(s):
    b, hq, d = s["q"].shape
    hkv = s["kv_heads"]
    table = s["block_table"].long()
    k = _gathered(s["k_pages"], table, s["k_scale"])
    q = s["q"].float().view(b, hkv, hq // hkv, d)
    scores = q @ k.transpose(-1, -2) / math.sqrt(d)
    keys = torch.arange(k.shape[2], device=k.device)
    seen = _visible((s["lens"].long() - 1)[:, None, None, None], keys, s["window"], s["sinks"])
    out = _softmax(scores, seen) @ _gathered(s["v_pages"], table, s["v_scale"])
    return out.view(b, hq, d).to(s["q"].dtype)


def _padded(x, cu, longest):
    """[batch, longest, heads, head dim] of a packed [tokens, heads, head dim] in fp32; what is past a sequence's end is not read by its own rows."""
    i = cu[:-1].long()[:, None] + torch.arange(longest, device=x.device)
    return x[i.clamp(max=x.shape[0] - 1)].float()


def _plain_prompt(s):
    t, hq, d = s["q"].shape
    hkv, cu_q, cu_k = s["kv_heads"], s["cu_q"], s["cu_k"]
    b = cu_q.shape[0] - 1
    q = _padded(s["q"], cu_q, s["max_q"]).view(b, s["max_q"], hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
    k, v = (_padded(x, cu_k, s["max_k"]).transpose(1, 2)[:, :, None] for x in (s["k"], s["v"]))
    scores = (q / math.sqrt(d)) @ k.transpose(-1, -2)
    n, m = cu_q.diff().long(), cu_k.diff().long()
    pos = (m - n)[:, None] + torch.arange(s["max_q"], device=q.device)
    seen = _visible(pos[:, None, None, :, None], torch.arange(s["max_k"], device=q.device), s["window"], s["sinks"])
    out = (_softmax(scores, seen) @ v).permute(0, 3, 1, 2, 4).reshape(b * s["max_q"], hq, d)
    row = torch.arange(t, device=q.device)
    which = torch.searchsorted(cu_q, row.to(torch.int32), right=True) - 1
    return out[which * s["max_q"] + row - cu_q.long()[which]].to(s["q"].dtype)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    d = case["head_dim"]
    group = case["q_heads"] // case["kv_heads"]
    if case["op"] == "qk_norm_rope":
        r = case["rotary"]
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.zeros((), dtype=torch.float64, device="cuda"))
        turn = turn * torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None]

        def heads(x, weight):
            x = x.double()
            if weight is not None:
                x = weight.double() * x / ((x * x).sum(-1, keepdim=True) / d + EPS).sqrt()
            z = torch.complex(x[..., : r // 2].contiguous(), x[..., r // 2 : r].contiguous()) * turn
            return torch.cat([z.real, z.imag, x[..., r:]], dim=-1)

        out = {"q": heads(s["q"], s["q_weight"]), "k": heads(s["k"], s["k_weight"])}
        if s["k_pages"] is not None:
            for name, x in (("k", out["k"]), ("v", s["v"].double())):
                flat = s[name + "_pages"].double().transpose(1, 2).reshape(-1, case["kv_heads"], d)
                if s[name + "_scale"] is not None:
                    x = (x / s[name + "_scale"].double()[None, :, None]).clamp(-F8_MAX, F8_MAX)
                flat[s["slots"]] = x
                out[name + "_pages"] = flat.view(-1, case["page"], case["kv_heads"], d).transpose(1, 2)
        return out

    def attend(q, k, v, first):
        """q [n, group, d], k and v [m, d] in 64 bits; the first query stands at position `first`."""
        n, m = q.shape[0], k.shape[0]
        out = torch.zeros_like(q)
        step = max(1, (1 << 27) // max(1, m * group))
        for i in range(0, n, step):
            at = first + torch.arange(i, min(n, i + step), device="cuda")[:, None]
            key = torch.arange(m, device="cuda")[None]
            hidden = key > at
            if case["window"] > 0:
                hidden |= (key <= at - case["window"]) & (key >= case["sinks"])
            logits = torch.einsum("ngd,md->gnm", q[i : i + step], k) * d**-0.5
            logits[:, hidden] = -math.inf
            out[i : i + step] = torch.einsum("gnm,md->ngd", torch.softmax(logits, -1).nan_to_num(0.0), v)
        return out

    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if case["op"] == "paged_attention":
        for b, n in enumerate(_lengths(case)):
            used = s["block_table"][b, : -(-n // case["page"])].long()
            for h in range(case["kv_heads"]):
                k, v = (s[x][:, h].view(torch.uint8 if case["cache"] == "fp8" else DTYPES[case["cache"]])[used].view(DTYPES[case["cache"]]) for x in ("k_pages", "v_pages"))
                k, v = (x.double().reshape(-1, d)[:n] for x in (k, v))
                if case["cache"] == "fp8":
                    k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
                rows = slice(h * group, (h + 1) * group)
                out[b, rows] = attend(s["q"][b : b + 1, rows].double(), k, v, n - 1)[0]
        return out
    q0 = k0 = 0
    for n in _lengths(case):
        m = n + case["past"]
        for h in range(case["kv_heads"]):
            rows = slice(h * group, (h + 1) * group)
            out[q0 : q0 + n, rows] = attend(s["q"][q0 : q0 + n, rows].double(), s["k"][k0 : k0 + m, h].double(), s["v"][k0 : k0 + m, h].double(), m - n)
        q0, k0 = q0 + n, k0 + m
    return out


# ---------------------------------------------------------------------------------------------------- what a pass has to do
def _size(name):
    return {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1, "none": 0}[name]


def _seen(pos, window, sinks):
    """How many keys the query at this position sees."""
    return pos + 1 if window <= 0 else min(pos + 1, window) + max(0, min(sinks, pos + 1 - window))


def work(case):
    hq, hkv, d, e = case["q_heads"], case["kv_heads"], case["head_dim"], _size(case["dtype"])
    if case["op"] == "qk_norm_rope":
        t = case["tokens"]
        moved = 2 * t * (hq + hkv) * d * e + t * 4 * (1 + case["rotary"])
        if case["cache"] != "none":
            moved += t * hkv * d * (e + 2 * _size(case["cache"])) + 8 * t
        return {"bytes": moved, "flops": t * (hq + hkv) * ((4 * d if case["norm"] else 0) + 3 * case["rotary"])}
    if case["op"] == "paged_attention":
        seen = [_seen(n - 1, case["window"], case["sinks"]) for n in _lengths(case)]
        return {"bytes": sum(seen) * hkv * d * 2 * _size(case["cache"]) + 2 * case["batch"] * hq * d * e, "flops": 4 * sum(seen) * hq * d}
    n = _lengths(case)
    seen = sum(_seen(case["past"] + i, case["window"], case["sinks"]) for x in n for i in range(x))
    return {"bytes": sum(n) * hq * d * 2 * e + 2 * (sum(n) + case["past"] * len(n)) * hkv * d * e, "flops": 4 * seen * hq * d}

