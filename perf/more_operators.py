"""Cases of the operators that answer many requests at once beside a decoder's quantized Linears: log probabilities of given tokens with the
entropy and the top alternatives (and their gradient), low-rank adapters of many requests added to a shared projection, and
attention of one new token of every sequence where groups of sequences share a long prefix.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}


# ---------------------------------------------------------------------------------------------------- cases
def _score(name, rows, vocab, dtype, top, allowed, ignored, gradient):
    """`allowed`: tokens of a row that a grammar leaves (0: all of them); `ignored`: share of rows without a token (padding)."""
    return dict(name=name, op="token_logprobs", rows=rows, vocab=vocab, dtype=dtype, top=top, allowed=allowed, ignored=ignored, gradient=gradient)


def _adapt(name, tokens, prompts, adapters, rank, width, out, dtype, without):
    """`prompts`: tokens stand in so many runs of one adapter each (0: every token has its own); `without`: share of them that have none."""
    return dict(name=name, op="lora_add", tokens=tokens, prompts=prompts, adapters=adapters, rank=rank, width=width, out=out, dtype=dtype, without=without)


def _shared(name, groups, each, prefix, longest, ragged, q_heads, kv_heads, head_dim, dtype, cache, page, window, sinks):
    """`groups` of `each` sequences share `prefix` tokens and have up to `longest` of their own behind them."""
    return dict(name=name, op="prefix_attention", groups=groups, each=each, prefix=prefix, longest=longest, ragged=ragged, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, dtype=dtype, cache=cache, page=page, window=window, sinks=sinks)  # fmt: skip


def listed():
    return [
        # the latest token of one sequence of the benchmark's decoder with five alternatives: a generated token's latency
        _score("score 1 x 128256 top 5", 1, 128256, "bf16", 5, 0, 0.0, False),
        # a decode batch with twenty alternatives
        _score("score 64 x 128256 top 20", 64, 128256, "bf16", 20, 0, 0.0, False),
        # two prompts of the benchmark's length scored for their perplexity
        _score("score 4096 x 128256", 4096, 128256, "bf16", 0, 0, 0.0, False),
        # a training step's loss: forward and the logits' gradient, some rows padding
        _score("gradient 2048 x 128256", 2048, 128256, "bf16", 0, 0, 0.1, True),
        # an odd vocabulary in fp32, where a grammar leaves few tokens
        _score("score 333 x 50257 fp32 9 allowed", 333, 50257, "fp32", 20, 9, 0.0, False),
        # one token of one request: the latency beside a projection
        _adapt("adapter 1 token", 1, 0, 4, 16, 4096, 4096, "bf16", 0.0),
        # a decode batch of many adapters beside a wide projection
        _adapt("adapter 64 tokens of 16", 64, 0, 16, 16, 4096, 14336, "bf16", 0.1),
        # the benchmark's prompts, an adapter each
        _adapt("adapter 8 prompts of 2048", 16384, 8, 8, 16, 4096, 4096, "bf16", 0.0),
        # prompts of odd lengths beside the down projection, a higher rank
        _adapt("adapter 1999 tokens rank 64", 1999, 5, 3, 64, 14336, 4096, "fp16", 0.2),
        # a few continuations of one prompt
        _shared("prefix 4 x (2048 + 128)", 1, 4, 2048, 128, False, 32, 8, 128, "bf16", "bf16", 16, 0, 0),
        # a serving batch behind one long instruction, cache in e4m3, ragged lengths
        _shared("prefix 61 x (8200 + 515) e4m3", 1, 61, 8200, 515, True, 32, 8, 128, "bf16", "fp8", 64, 0, 0),
        # two documents, many questions about each
        _shared("prefix 2 of 64 x (32768 + 300)", 2, 64, 32768, 300, True, 32, 8, 128, "bf16", "bf16", 64, 0, 0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["token_logprobs", "lora_add", "prefix_attention"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "token_logprobs":
        vocab = _log(rng, 500, 260000)
        rows = _log(rng, 1, min(8192, 200000000 // vocab))
        c = _score("", rows, vocab, rng.choice([dtype, dtype, "fp32"]), rng.choice([0, 1, 5, 20, 32]), rng.choice([0, 0, 0, 3, 200]), rng.choice([0.0, 0.0, 0.3]),
                   rng.random() < 0.3)  # fmt: skip
    elif op == "lora_add":
        tokens = _log(rng, 1, 8192)
        prompts = rng.choice([0, _log(rng, 1, min(32, tokens))]) if tokens <= 256 else _log(rng, 1, 32)
        width, out = (8 * _log(rng, 64, 1024) for _ in range(2))
        c = _adapt("", tokens, prompts, _log(rng, 1, 32), rng.choice([8, 16, 24, 32, 64, 128]), width, out, dtype, rng.choice([0.0, 0.0, 0.3]))
    else:
        hq, hkv = rng.choice([(32, 8), (12, 12), (16, 2), (8, 1), (40, 8)])
        dim = rng.choice([64, 96, 128])
        prefix, longest = _log(rng, 16, 30000), _log(rng, 1, 1200)
        groups = rng.choice([1, 1, 1, 2, 3])
        each = _log(rng, 1, max(1, min(64, 3000000 // (groups * (prefix // 8 + longest)))))
        window, sinks = rng.choice([(0, 0), (0, 0), (0, 0), (1024, 4), (4096, 1)])
        c = _shared("", groups, each, prefix, longest, rng.random() < 0.7, hq, hkv, dim, dtype, rng.choice([dtype, "fp8"]), rng.choice([16, 24, 32, 64, 128]), window, sinks)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prefixes(case):
    """Lengths of the groups' prefixes: a little shorter from group to group."""
    return [max(1, case["prefix"] - (case["prefix"] * i) // (8 * case["groups"])) for i in range(case["groups"])]


def _owns(case):
    """Tokens of their own of a group's sequences, the longest first."""
    n, each = case["longest"], case["each"]
    return [max(1, n - (n * i) // each) if case["ragged"] else n for i in range(each)]


def _pages(g, pages, case):
    """A pool of keys or values, made in parts so that a long cache needs no fp32 copy of itself."""
    out = torch.empty((pages, case["kv_heads"], case["page"], case["head_dim"]), dtype=DTYPES[case["cache"]], device="cuda")
    part = max(1, (1 << 27) // out[0].numel())
    for i in range(0, pages, part):
        out[i : i + part] = _randn(g, out[i : i + part].shape, torch.float32).to(out.dtype)
    return out


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "token_logprobs":
        n, v = case["rows"], case["vocab"]
        s["tokens"] = torch.randint(0, v, (n,), generator=g, device="cuda")
        logits = torch.empty((n, v), dtype=dt, device="cuda")
        part = max(1, (1 << 27) // v)
        for i in range(0, n, part):  # a model's logits: the token that follows stands out in most rows
            x = _randn(g, logits[i : i + part].shape, torch.float32, 2.5)
            x.scatter_add_(1, s["tokens"][i : i + part, None], torch.rand((x.shape[0], 1), generator=g, device="cuda") * 16)
            if case["allowed"]:  # every so many-th token, and the one that follows, which an entry of zero leaves as it is
                step = max(1, v // case["allowed"])
                shut = (torch.arange(v, device="cuda") + torch.arange(x.shape[0], device="cuda")[:, None]) % step != 0
                shut.scatter_(1, s["tokens"][i : i + part, None], False)
                x.masked_fill_(shut, -math.inf)
            logits[i : i + part] = x.to(dt)
        s["logits"] = logits
        if case["ignored"]:
            s["tokens"] = torch.where(torch.rand(n, generator=g, device="cuda") < case["ignored"], -100, s["tokens"])
        if case["gradient"]:
            s["logits"].requires_grad_(True)
            s["d_logprobs"], s["d_entropy"] = _randn(g, (n,), torch.float32), _randn(g, (n,), torch.float32, 0.1)
    elif case["op"] == "lora_add":
        t, n, r, k, out = (case[x] for x in ("tokens", "adapters", "rank", "width", "out"))
        s["x"], s["y"] = _randn(g, (t, k), dt), _randn(g, (t, out), dt)
        s["a"], s["b"] = _randn(g, (n, r, k), dt, k**-0.5), _randn(g, (n, out, r), dt, 0.05)
        s["scale"] = torch.rand(n, generator=g, device="cuda") * 2 + 0.5
        runs = case["prompts"] or t
        which = torch.randint(0, n, (runs,), generator=g, device="cuda")
        which = torch.where(torch.rand(runs, generator=g, device="cuda") < case["without"], n, which)
        if case["prompts"]:
            ends = torch.rand(runs - 1, generator=g, device="cuda").mul(t).long().sort().values
            which = which[torch.searchsorted(ends, torch.arange(t, device="cuda"), right=True)]
        # the rows of each adapter: made once a step, for all projections of all layers
        order = torch.sort(which, stable=True)
        s["starts"] = torch.searchsorted(order.values, torch.arange(n + 1, device="cuda")).to(torch.int32)
        s["rows"] = order.indices[: int(s["starts"][-1])].to(torch.int32)
    else:
        page, hkv, d, groups, each = case["page"], case["kv_heads"], case["head_dim"], case["groups"], case["each"]
        first, behind = _prefixes(case), _owns(case)
        b = groups * each
        lens = [p + n for p in first for n in behind]
        per_prefix, per = -(-max(first) // page), -(-max(lens) // page)
        own_first = min(first) // page  # the first page that holds a token of a sequence's own
        pages = groups * per_prefix + b * (per - own_first) + 1
        s["q"] = _randn(g, (b, case["q_heads"], d), dt, 1.5)
        s["k_pages"], s["v_pages"] = _pages(g, pages, case), _pages(g, pages, case)
        order = torch.randperm(pages - 1, generator=g, device="cuda").to(torch.int32)
        s["prefix_table"] = order[: groups * per_prefix].view(groups, per_prefix)
        s["block_table"] = torch.zeros((b, per), dtype=torch.int32, device="cuda")
        s["block_table"][:, own_first:] = order[groups * per_prefix :].view(b, per - own_first)
        s["prefix_lens"], s["lens"], s["groups_at"] = _int32(first), _int32(lens), _int32([i * each for i in range(groups + 1)])
        s["own_first"] = own_first
        s["k_scale"] = s["v_scale"] = None
        if case["cache"] == "fp8":
            s["k_scale"], s["v_scale"] = (torch.rand(hkv, generator=g, device="cuda") * 0.5 + 0.75 for _ in range(2))
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def run(s):
    if s["op"] == "token_logprobs":
        return _own_score(s) if own else _plain_score(s)
    if s["op"] == "lora_add":
        return _own_adapt(s) if own else _plain_adapt(s)
    return _own_shared(s) if own else _plain_shared(s)


def _scored(logprobs, entropy, top_logprobs, top_ids, d_logits):
    out = {"logprobs": logprobs, "entropy": entropy}
    if top_ids is not None:
        out.update(top_logprobs=top_logprobs, top_ids=top_ids)
    if d_logits is not None:
        out["d_logits"] = d_logits
    return out


def _own_score(s):
    from fms_model_optimizer_b200 import ops

    logprobs, entropy, top_logprobs, top_ids = ops.token_logprobs(s["logits"], s["tokens"], top=s["top"])
    grad = None
    if s["gradient"]:
        (grad,) = torch.autograd.grad((logprobs, entropy), s["logits"], (s["d_logprobs"], s["d_entropy"]))
    return _scored(logprobs.detach(), entropy.detach(), *((top_logprobs, top_ids) if s["top"] else (None, None)), grad)


def _own_adapt(s):
    from fms_model_optimizer_b200 import ops

    return ops.lora_add_(s["y"], s["x"], s["a"], s["b"], s["rows"], s["starts"], s["scale"])


def _own_shared(s):
    from fms_model_optimizer_b200 import ops

    return ops.prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["prefix_table"], s["prefix_lens"], s["groups_at"], s["block_table"], s["lens"],
                                window=s["window"], sinks=s["sinks"], k_scale=s["k_scale"], v_scale=s["v_scale"])  # fmt: skip


def _plain_top(x, count):
    """Ids of the largest values of each row, ties to the lowest: one order of (value, id) in 64 bits."""
    bits = x.contiguous().view(torch.int32).long()
    keys = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    keys = keys * (1 << 32) + (x.shape[-1] - 1 - torch.arange(x.shape[-1], device=x.device))
    return x.shape[-1] - 1 - keys.topk(count, dim=-1, sorted=True).values.remainder(1 << 32)


def _plain_score(s):
    x, tokens = s["logits"].detach().float(), s["tokens"]
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    log_p = x - total.log()
    p = e / total
    known = tokens >= 0
    logprobs = torch.where(known, log_p.gather(1, tokens.clamp(min=0)[:, None])[:, 0], 0.0)
    p_log_p = torch.where(p > 0, p * log_p, 0.0)
    entropy = -p_log_p.sum(-1)
    top_logprobs = top_ids = grad = None
    if s["top"]:
        top_ids = _plain_top(s["logits"].detach().float(), s["top"])
        top_logprobs = log_p.gather(1, top_ids)
    if s["gradient"]:
        dl = torch.where(known, s["d_logprobs"], 0.0)[:, None]
        grad = -dl * p - s["d_entropy"][:, None] * (p_log_p + p * entropy[:, None])
        grad = grad.scatter_add(1, tokens.clamp(min=0)[:, None], dl).to(s["logits"].dtype)
    return _scored(logprobs, entropy, top_logprobs, top_ids, grad)


def _plain_adapt(s):
    rows, n, r = s["rows"].long(), s["adapters"], s["rank"]
    which = torch.searchsorted(s["starts"][1:], torch.arange(rows.shape[0], device=rows.device, dtype=torch.int32), right=True)
    low = s["x"][rows].float() @ s["a"].float().flatten(0, 1).t()  # by every adapter; all but a row's own are struck out
    mine = torch.arange(n * r, device=rows.device) // r == which[:, None]
    low = torch.where(mine, low * s["scale"][which][:, None], 0.0)
    more = low @ s["b"].float().transpose(1, 2).flatten(0, 1)
    s["y"][rows] = (s["y"][rows].float() + more).to(s["y"].dtype)
    return s["y"]


def _gathered(pages, table, scale):
    """[sequences, kv heads, keys, head dim] in fp32."""
    table = table.long()
    x = (pages.view(torch.uint8)[table].view(pages.dtype) if pages.dtype == torch.float8_e4m3fn else pages[table]).float()
    x = x.transpose(1, 2).flatten(2, 3)
    return x if scale is None else x * scale[:, None, None]


def _visible(pos, keys, window, sinks):
    seen = keys <= pos
    return seen & ((keys > pos - window) | (keys < sinks)) if window > 0 else seen


def _plain_shared(s):
    b, hq, d = s["q"].shape
    hkv, groups, each = s["kv_heads"], s["groups"], s["each"]
    q = s["q"].float().view(groups, each, hkv, hq // hkv, d) / math.sqrt(d)
    pos = (s["lens"].long() - 1).view(groups, each, 1, 1, 1)
    first = s["prefix_lens"].long().view(groups, 1, 1, 1, 1)
    # every group's rows against its prefix, every sequence's against its own keys
    kp, vp = (_gathered(s[x + "_pages"], s["prefix_table"], s[x + "_scale"])[:, None] for x in "kv")
    ko, vo = (_gathered(s[x + "_pages"], s["block_table"][:, s["own_first"] :], s[x + "_scale"]).unflatten(0, (groups, each)) for x in "kv")
    key = torch.arange(kp.shape[3], device=q.device)
    seen = _visible(pos, key, s["window"], s["sinks"]) & (key < first)
    rows = q.transpose(1, 2).flatten(2, 3)  # [groups, kv heads, rows, d]
    xp = (rows @ kp[:, 0].transpose(-1, -2)).unflatten(2, (each, hq // hkv)).transpose(1, 2).masked_fill(~seen, -math.inf)
    key = torch.arange(ko.shape[3], device=q.device) + s["own_first"] * s["page"]
    seen = _visible(pos, key, s["window"], s["sinks"]) & (key >= first)
    xo = (q @ ko.transpose(-1, -2)).masked_fill(~seen, -math.inf)
    top = torch.maximum(xp.amax(-1, keepdim=True), xo.amax(-1, keepdim=True))
    wp, wo = (xp - top).exp(), (xo - top).exp()
    total = wp.sum(-1, keepdim=True) + wo.sum(-1, keepdim=True)
    shared = (wp.transpose(1, 2).flatten(2, 3) @ vp[:, 0]).unflatten(2, (each, hq // hkv)).transpose(1, 2)
    return ((shared + wo @ vo) / total).reshape(b, hq, d).to(s["q"].dtype)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "token_logprobs":
        return _exact_score(case, s)
    if case["op"] == "lora_add":
        y = s["y"].double()
        at = s["starts"].tolist()
        for i in range(case["adapters"]):
            rows = s["rows"][at[i] : at[i + 1]].long()
            y[rows] += s["scale"][i].double() * torch.einsum("tk,rk,nr->tn", s["x"][rows].double(), s["a"][i].double(), s["b"][i].double())
        return y
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    d, page, heads = case["head_dim"], case["page"], case["q_heads"] // case["kv_heads"]
    raw = {x: s[x + "_pages"].view(torch.uint8) if case["cache"] == "fp8" else s[x + "_pages"] for x in "kv"}
    for b, n in enumerate(s["lens"].tolist()):
        group = b // case["each"]
        key = torch.arange(n, device="cuda")
        if case["window"]:
            key = key[(key > n - 1 - case["window"]) | (key < case["sinks"])]
        mine = key >= s["prefix_lens"][group]
        at = torch.where(mine, s["block_table"][b][key // page], s["prefix_table"][group][(key // page).clamp(max=s["prefix_table"].shape[1] - 1)]).long()
        k, v = (raw[x][at, :, key % page].view(DTYPES[case["cache"]]).double() for x in "kv")  # [keys, kv heads, d]
        if case["cache"] == "fp8":
            k, v = k * s["k_scale"].double()[:, None], v * s["v_scale"].double()[:, None]
        q = s["q"][b].double().view(case["kv_heads"], heads, d)
        weights = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) * d**-0.5, -1)
        out[b] = torch.einsum("hgn,nhd->hgd", weights, v).reshape(-1, d)
    return out


def _exact_score(case, s):
    n, v = case["rows"], case["vocab"]
    out = {"logprobs": torch.zeros(n, dtype=torch.float64, device="cuda"), "entropy": torch.zeros(n, dtype=torch.float64, device="cuda")}
    if case["top"]:
        out["top_logprobs"] = torch.zeros((n, case["top"]), dtype=torch.float64, device="cuda")
        out["top_ids"] = torch.zeros((n, case["top"]), dtype=torch.int64, device="cuda")
    if case["gradient"]:
        out["d_logits"] = torch.zeros((n, v), dtype=torch.float64, device="cuda")
    part = max(1, (1 << 25) // v)
    for i in range(0, n, part):
        rows = slice(i, min(n, i + part))
        x, tokens = s["logits"][rows].detach().double(), s["tokens"][rows]
        log_p = x - torch.logsumexp(x, -1, keepdim=True)
        at = torch.arange(x.shape[0], device="cuda")
        out["logprobs"][rows] = torch.where(tokens < 0, 0.0, log_p[at, tokens.clamp(min=0)])
        out["entropy"][rows] = torch.special.entr(log_p.exp()).sum(-1)
        if case["top"]:
            ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, : case["top"]]
            out["top_ids"][rows], out["top_logprobs"][rows] = ids, log_p[at[:, None], ids]
        if case["gradient"]:
            grad = torch.zeros_like(x)
            grad[at, tokens.clamp(min=0)] = torch.where(tokens < 0, 0.0, s["d_logprobs"][rows].double())
            grad -= log_p.exp() * grad.sum(-1, keepdim=True)
            grad += s["d_entropy"][rows, None].double() * (torch.special.entr(log_p.exp()) - log_p.exp() * out["entropy"][rows, None])
            out["d_logits"][rows] = grad
    return out


# ---------------------------------------------------------------------------------------------------- what a pass has to do
def _size(name):
    return {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}[name]


def work(case):
    e = _size(case["dtype"])
    if case["op"] == "token_logprobs":
        n = case["rows"] * case["vocab"]
        moved = n * e + case["rows"] * (8 + 4 + 4 + 12 * case["top"])
        if case["gradient"]:  # the gradient needs the sums of the whole row first, so it reads the logits again
            moved += 2 * n * e + case["rows"] * 8
        return {"bytes": moved, "flops": n * (13 if case["gradient"] else 5)}
    if case["op"] == "lora_add":
        t, r, k, out = case["tokens"] * (1 - case["without"]), case["rank"], case["width"], case["out"]
        used = min(case["adapters"], case["prompts"] or case["tokens"])
        return {"bytes": int((t * (k + 2 * out) + used * r * (k + out)) * e), "flops": int(2 * t * r * (k + out))}
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    keys = seen = 0
    for p in _prefixes(case):
        lens = [p + n for n in _owns(case)]
        start = [max(0, n - case["window"]) if case["window"] else 0 for n in lens]
        some = [min(case["sinks"], x) for x in start]
        seen += sum(n - x + f for n, x, f in zip(lens, start, some))
        low, first = min(min(start), p), min(max(some), p)
        keys += p - low + min(first, low) + sum(n - max(x, p) + max(0, f - p) for n, x, f in zip(lens, start, some))
    return {"bytes": keys * hkv * d * 2 * _size(case["cache"]) + 2 * case["groups"] * case["each"] * hq * d * e, "flops": 4 * seen * hq * d}
