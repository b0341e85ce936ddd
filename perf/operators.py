"""The operators of the latent (MLA) cache as data and functions: what a serving or sampling loop of the MLA layer runs.

  append     RMSNorm of the latent part and rotation of the rotary part of new tokens, written into cache pages (bf16 or fp8)
  gather     the rows of the sequences' pages, in order, back as bf16 (for the expanded form of a prompt behind a cached prefix)
  absorb     the products around the attention: queries into the latent space (and their rotation), results out of it
  attention  one or a few new tokens a sequence against its cached rows, causal
  tree       the same for a tree of drafted tokens, whose mask is a word of bits a token

`own` says who computes: False the plain form below, elementary torch operations in 32 bits, True the framework's operators.
Sizes are those of DeepSeek-V2-Lite's layer: 512 latent, 64 rotary, 128 nope and 128 value features; 16 heads, or 128 as in the operator matrix of
the benchmark. Imported with the root of the tree under measurement as the working folder.
"""

import math
import os
import random
import sys

import torch

own = False

LATENT, ROPE, NOPE, VALUE = 512, 64, 128, 128
SCALE = (NOPE + ROPE) ** -0.5
EPS = 1e-6
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
POSITIONS = 16384  # of the rotary tables


def _operators():
    package = os.path.join(os.getcwd(), "pith-train_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from pithtrain_amd.operators.mla import latent

    return latent


# ---------------------------------------------------------------------------------------------
# Cases


def _append(name, tokens, run, cache, page, weight="bf16"):
    """`run` consecutive tokens a sequence: 1 while answering, the prompt's length while reading it."""
    return {"name": name, "kind": "append", "tokens": tokens, "run": run, "cache": cache, "page": page, "weight": weight}


def _gather(name, b, longest, least, cache, page):
    return {"name": name, "kind": "gather", "b": b, "longest": longest, "least": least, "cache": cache, "page": page}


def _absorb(name, side, tokens, h):
    return {"name": name, "kind": "absorb", "side": side, "tokens": tokens, "h": h}


def _attention(name, kind, b, h, q, longest, least, cache, page, even=True):
    """`q` new tokens a sequence (even) or 1 .. q; cached lengths, new tokens included, from least * longest to longest."""
    return {"name": name, "kind": kind, "b": b, "h": h, "q": q, "longest": longest, "least": least, "cache": cache, "page": page, "even": even}


def listed():
    return [
        # One step of 32 sequences that are being answered: their new rows go into 32 pages, quantised.
        _append("append_step_fp8", 32, 1, "fp8", 64),
        # A prompt of 8192 tokens is read in: the cache as bf16.
        _append("append_prompt", 8192, 8192, "bf16", 64),
        # A prefix of odd length comes back for the expanded form of the prompt behind it.
        _gather("gather_prefix", 1, 1021, 1.0, "bf16", 64),
        # The prefixes of a batch of prompts from an fp8 cache.
        _gather("gather_batch_fp8", 16, 8192, 0.25, "fp8", 64),
        # The queries of one step of 32 sequences, 16 heads: all latency and weights.
        _absorb("absorb_query_step", "query", 32, 16),
        # Results of a wide layer (128 heads) for a few hundred tokens.
        _absorb("absorb_value_wide", "value", 509, 128),
        # The smallest step: one sequence of a few hundred tokens.
        _attention("decode_small", "attention", 1, 16, 1, 517, 1.0, "bf16", 64),
        # An ordinary step: 32 sequences of very different lengths.
        _attention("decode_batch", "attention", 32, 16, 1, 8192, 0.1, "bf16", 64),
        # Long contexts from an fp8 cache: the largest by bytes.
        _attention("decode_long_fp8", "attention", 8, 16, 1, 131072, 0.5, "fp8", 64),
        # 128 heads share every cached row: as much arithmetic as memory.
        _attention("decode_128_heads", "attention", 32, 128, 1, 8192, 0.25, "bf16", 64),
        # A small tree of drafts for four sequences.
        _attention("tree_small_fp8", "tree", 4, 16, 8, 1500, 0.5, "fp8", 64),
        # Large trees of different sizes for a batch: the largest by arithmetic.
        _attention("tree_batch", "tree", 16, 16, 48, 16384, 0.25, "bf16", 16, even=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _draw_any(rng):
    kind = rng.choice(["append", "gather", "absorb", "attention", "attention", "attention", "tree", "tree"])
    cache, page = rng.choice(["bf16", "fp8"]), rng.choice([16, 32, 64, 64, 128])
    least = rng.choice([0.05, 0.3, 0.7, 1.0])
    if kind == "append":
        tokens = _log_int(rng, 1, 16384)
        case = _append("", tokens, rng.choice([1, tokens]) if tokens <= 256 else _log_int(rng, 64, tokens), cache, page, rng.choice(["bf16", "fp32"]))
    elif kind == "gather":
        case = _gather("", _log_int(rng, 1, 64), _log_int(rng, 1, 32768), least, cache, page)
    elif kind == "absorb":
        case = _absorb("", rng.choice(["query", "value"]), _log_int(rng, 1, 4096), rng.choice([4, 16, 16, 128]))
    elif kind == "attention":
        q = rng.choice([1, 1, 1, 2, 3, rng.randint(4, 64)])
        case = _attention("", kind, _log_int(rng, 1, 128), rng.choice([4, 16, 16, 128]), q, _log_int(rng, 1, 131072), least, cache, page, rng.random() < 0.5)
    else:
        case = _attention("", kind, _log_int(rng, 1, 64), rng.choice([4, 16, 16, 128]), rng.randint(2, 64), _log_int(rng, 1, 65536), least, cache, page, rng.random() < 0.5)
    case.pop("name")
    return case


def draw(rng):
    """One more case of these ranges; none costs more than the largest listed ones."""
    most = {m: max(work(c)[m] for c in listed()) for m in ("bytes", "flops")}
    while True:
        case = _draw_any(rng)
        w = work(case)
        if any(w[m] > most[m] for m in most):
            continue
        if case["kind"] in ("attention", "tree"):  # what the plain form lays out: padded keys and scores in 32 bits
            keys = case["b"] * max(_lengths(case))
            if keys * (LATENT + ROPE) * 4 > 6 << 30 or keys * max(_counts(case)) * case["h"] * 4 > 6 << 30:
                continue
        return case


def _counts(case):
    """New tokens of each sequence."""
    b, q = case["b"], case.get("q", 0)
    return [q if case.get("even", True) else 1 + (7 * i + q - 1) % q for i in range(b)]


def _lengths(case):
    """Cached rows of each sequence, its new tokens among them: spread evenly between the shortest and the longest."""
    spread = [(i * 0.6180339887498949) % 1.0 for i in range(case["b"])]
    least, longest = case["least"], case["longest"]
    return [max(n, 1, int(round(longest * (1.0 - (1.0 - least) * f)))) for n, f in zip(_counts(case), spread)]


def _row_bytes(case):
    return 2 * (LATENT + ROPE) if case["cache"] == "bf16" else LATENT + 2 * ROPE + 4


def work(case):
    kind = case["kind"]
    if kind == "append":
        t = case["tokens"]
        return {"bytes": t * (2 * (LATENT + ROPE) + 4 * ROPE + 16 + _row_bytes(case)) + LATENT * (2 if case["weight"] == "bf16" else 4), "flops": t * (4 * LATENT + 6 * ROPE)}
    if kind == "gather":
        rows = sum(_lengths(case))
        return {"bytes": rows * (_row_bytes(case) + 2 * (LATENT + ROPE)), "flops": 0 if case["cache"] == "bf16" else rows * LATENT}
    if kind == "absorb":
        t, h = case["tokens"], case["h"]
        n_in, n_out = (NOPE + ROPE, LATENT + ROPE) if case["side"] == "query" else (LATENT, VALUE)
        tables = t * (4 * ROPE + 8) if case["side"] == "query" else 0
        return {"bytes": 2 * t * h * (n_in + n_out) + 2 * h * NOPE * LATENT + tables, "flops": 2 * t * h * NOPE * LATENT}
    counts, lengths, h = _counts(case), _lengths(case), case["h"]
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(counts, lengths))
    t = sum(counts)
    return {"bytes": sum(lengths) * _row_bytes(case) + t * h * (2 * (LATENT + ROPE) + 2 * LATENT + 4), "flops": 2 * h * pairs * (2 * LATENT + ROPE)}


# ---------------------------------------------------------------------------------------------
# What the program has in hand


def _tables(g, dev):
    angle = torch.arange(POSITIONS, device=dev, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(0, ROPE, 2, device=dev, dtype=torch.float64) / ROPE)
    angle = torch.cat((angle, angle), 1)
    return angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)


def _cache(case, pages, g, dev):
    """Pages full of rows as they are after the norm (features of different size, a few tokens much larger) and the rotation."""
    page = case["page"]
    latent = torch.randn(pages, page, LATENT, generator=g, device=dev) * (0.5 + torch.rand(LATENT, generator=g, device=dev))
    k_pe = (2.0 * torch.randn(pages, page, ROPE, generator=g, device=dev)).to(torch.bfloat16)
    if case["cache"] == "bf16":
        return latent.to(torch.bfloat16), k_pe, None
    scale = latent.abs().amax(-1) / FP8_MAX
    return (latent / scale[..., None]).clamp(-FP8_MAX, FP8_MAX).to(FP8), k_pe, scale


def _page_table(case, lengths, g, dev):
    """Pages of each sequence in an order of their own; what a row of the table does not need points to a page of somebody else."""
    need = [-(-length // case["page"]) for length in lengths]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = order[torch.randint(0, pages, (len(need), max(need)), generator=g, device=dev)]
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at : at + n]
        at += n
    return table.contiguous(), pages


def _offsets(counts, dev):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=dev)


def _tree_words(case, seed):
    """A random tree of drafts a sequence: every draft has a parent among the earlier ones or none; it sees its ancestors and itself."""
    rng, words = random.Random(seed), []
    for n in _counts(case):
        mine = []
        for i in range(n):
            parent = rng.randint(max(-1, i - 8), i - 1)
            mine.append((mine[parent] if parent >= 0 else 0) | 1 << i)
        words += [w - (1 << 64) if w >> 63 else w for w in mine]
    return words


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    kind = case["kind"]
    bf16 = lambda *s, std=1.0: (std * torch.randn(*s, generator=g, device=dev)).to(torch.bfloat16)  # noqa: E731
    state = {"kind": kind}
    if kind == "append":
        t, page, run = case["tokens"], case["page"], case["run"]
        runs = -(-t // run)
        per_run = -(-run // page)
        pages = runs * per_run + 2
        order = torch.randperm(pages, generator=g, device=dev)[: runs * per_run].view(runs, per_run)
        i = torch.arange(t, device=dev)
        at = i % run if run > 1 else torch.randint(0, page, (t,), generator=g, device=dev)
        state["latent"], state["k_pe"], state["scale"] = _cache(case, pages, g, dev)
        state["slots"] = order[i // run, at // page] * page + at % page
        state["positions"] = at if run > 1 else torch.randint(0, POSITIONS, (t,), generator=g, device=dev)
        state["kv_a"] = bf16(t, LATENT + ROPE, std=1.5)
        state["weight"] = (1.0 + 0.2 * torch.randn(LATENT, generator=g, device=dev)).to(torch.bfloat16 if case["weight"] == "bf16" else torch.float32)
        state["cos"], state["sin"] = _tables(g, dev)
        return state
    if kind == "absorb":
        t, h = case["tokens"], case["h"]
        state["side"] = case["side"]
        state["weight"] = bf16(h * (NOPE + VALUE), LATENT, std=LATENT**-0.5)
        if case["side"] == "value":
            state["o_latent"] = bf16(t, h, LATENT, std=0.3)
            return state
        state["q"] = bf16(t, h, NOPE + ROPE)
        state["cos"], state["sin"] = _tables(g, dev)
        state["positions"] = torch.randint(0, POSITIONS, (t,), generator=g, device=dev)
        return state
    lengths = _lengths(case)
    state["page_table"], pages = _page_table(case, lengths, g, dev)
    state["latent"], state["k_pe"], state["scale"] = _cache(case, pages, g, dev)
    if kind == "gather":
        state["rows"] = sum(lengths)
        state["cu_rows"] = _offsets(lengths, dev)
        return state
    counts, h = _counts(case), case["h"]
    t = sum(counts)
    state["most"] = max(counts)
    state["q_latent"], state["q_pe"] = bf16(t, h, LATENT, std=0.6), bf16(t, h, ROPE)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
    state["cu_q"] = _offsets(counts, dev)
    state["tree"] = torch.tensor(_tree_words(case, seed), dtype=torch.int64, device=dev) if kind == "tree" else None
    return state


# ---------------------------------------------------------------------------------------------
# The plain form


def _rotated(x, cos, sin):
    """Pairs (2j, 2j + 1) of the last dimension become (j, j + ROPE / 2) and are rotated; cos, sin broadcast against x."""
    x = torch.cat((x[..., 0::2], x[..., 1::2]), -1)
    half = ROPE // 2
    return x * cos + torch.cat((-x[..., half:], x[..., :half]), -1) * sin


def _plain_append(s):
    x = s["kv_a"].float()
    c = x[:, :LATENT]
    c = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    pe = _rotated(x[:, LATENT:], s["cos"][s["positions"]].float(), s["sin"][s["positions"]].float())
    s["k_pe"].view(-1, ROPE)[s["slots"]] = pe.to(torch.bfloat16)
    if s["scale"] is None:
        s["latent"].view(-1, LATENT)[s["slots"]] = c.to(torch.bfloat16)
        return
    scale = c.abs().amax(-1) / FP8_MAX
    s["scale"].view(-1)[s["slots"]] = scale
    q = (c / scale[:, None]).clamp(-FP8_MAX, FP8_MAX).to(FP8)
    s["latent"].view(torch.uint8).view(-1, LATENT)[s["slots"]] = q.view(torch.uint8)


def _pages(s):
    """Latent and rotary rows of the pages of every table row, [b, most rows, features] in 32 bits."""
    table = s["page_table"].long()
    latent, k_pe = s["latent"].view(torch.uint8)[table].view(s["latent"].dtype).float(), s["k_pe"][table].float()
    if s["scale"] is not None:
        latent = latent * s["scale"][table][..., None]
    return latent.flatten(1, 2), k_pe.flatten(1, 2)


def _plain_gather(s):
    rows = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["cu_rows"], rows, right=True) - 1
    at = rows - s["cu_rows"][seq]
    page = s["latent"].shape[1]
    slot = s["page_table"][seq, at // page].long() * page + at % page
    latent = s["latent"].view(torch.uint8).view(len(s["latent"]) * page, -1)[slot].view(s["latent"].dtype).float()
    if s["scale"] is not None:
        latent = latent * s["scale"].view(-1)[slot][:, None]
    return latent.to(torch.bfloat16), s["k_pe"].view(-1, ROPE)[slot]


def _plain_absorb(s):
    if s["side"] == "value":
        h = s["o_latent"].shape[1]
        w = s["weight"].float().view(h, NOPE + VALUE, LATENT)[:, NOPE:]
        return torch.matmul(s["o_latent"].float().transpose(0, 1), w.transpose(1, 2).contiguous()).transpose(0, 1).to(torch.bfloat16).contiguous()
    q = s["q"].float()
    h = q.shape[1]
    w = s["weight"].float().view(h, NOPE + VALUE, LATENT)[:, :NOPE].contiguous()
    cos, sin = s["cos"][s["positions"]].float()[:, None], s["sin"][s["positions"]].float()[:, None]
    q_latent = torch.matmul(q[..., :NOPE].transpose(0, 1), w).transpose(0, 1)
    return q_latent.to(torch.bfloat16).contiguous(), _rotated(q[..., NOPE:], cos, sin).to(torch.bfloat16)


def _plain_attention(s):
    latent, k_pe = _pages(s)
    b, keys, _ = latent.shape
    t, h, _ = s["q_latent"].shape
    most, cu_q = s["most"], s["cu_q"].long()
    counts, lengths = cu_q[1:] - cu_q[:-1], s["lengths"].long()
    i = torch.arange(most, device="cuda")
    token = (cu_q[:-1, None] + i).clamp(max=t - 1)  # [b, most]; what lies behind a sequence's own tokens is left out below
    q = torch.cat((s["q_latent"], s["q_pe"]), -1).float()[token].flatten(1, 2)
    score = torch.matmul(q, torch.cat((latent, k_pe), -1).transpose(1, 2)) * SCALE
    before = (lengths - counts)[:, None, None]  # keys in front of the new tokens
    j = torch.arange(keys, device="cuda")
    if s["tree"] is None:
        seen = j <= before + i[None, :, None]
    else:
        bit = (j - before).clamp(0, 63)
        seen = (j < before) | ((s["tree"][token][..., None] >> bit) & 1).bool()
    seen = seen & (j < lengths[:, None, None])
    score = score.view(b, most, h, keys).masked_fill(~seen[:, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(1, 2), latent).view(b, most, h, LATENT) / torch.where(total == 0, 1.0, total)
    lse = ((top + torch.log(total)) * (1.0 / math.log(2.0)))[..., 0]
    all_tokens = torch.arange(t, device="cuda")
    seq = torch.searchsorted(cu_q, all_tokens, right=True) - 1
    mine = all_tokens - cu_q[seq]
    return o[seq, mine].to(torch.bfloat16), lse[seq, mine].t().contiguous()


def run(state):
    s = state
    kind = s["kind"]
    if own:
        ops = _operators()
        cache = None if kind == "absorb" else ops.LatentCache(s["latent"], s["k_pe"], s["scale"])
        if kind == "append":
            ops.latent_cache_append(s["kv_a"], s["weight"], s["cos"], s["sin"], s["positions"], s["slots"], cache, EPS)
        elif kind == "gather":
            return ops.latent_cache_gather(cache, s["page_table"], s["cu_rows"], s["rows"])
        elif kind == "absorb" and s["side"] == "query":
            return ops.absorb_query(s["q"], s["weight"], s["cos"], s["sin"], s["positions"])
        elif kind == "absorb":
            return ops.absorb_value(s["o_latent"], s["weight"])
        else:
            return ops.latent_attention(s["q_latent"], s["q_pe"], cache, s["page_table"], s["lengths"], s["cu_q"], SCALE, s["tree"])
    elif kind == "append":
        _plain_append(s)
    elif kind == "gather":
        return _plain_gather(s)
    elif kind == "absorb":
        return _plain_absorb(s)
    else:
        return _plain_attention(s)
    return {k: s[k] for k in ("latent", "k_pe", "scale")}  # the cache with its new rows


# ---------------------------------------------------------------------------------------------
# The definition in 64 bits


def _turned(x, cos, sin):
    """The rotation as complex numbers: feature pairs (2j, 2j + 1) times cos_j + i sin_j, real parts first."""
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], ROPE // 2, 2).contiguous()) * torch.complex(cos[..., : ROPE // 2].contiguous(), sin[..., : ROPE // 2].contiguous())
    return torch.cat((z.real, z.imag), -1)


def _exact_rows(s, seq, length):
    """Latent and rotary rows 0 .. length-1 of one sequence."""
    page = s["latent"].shape[1]
    at = torch.arange(length, device="cuda")
    p, r = s["page_table"][seq, at // page].long(), at % page
    c = s["latent"].to(torch.float32)[p, r].double()
    if s["scale"] is not None:
        c = c * s["scale"][p, r].double()[:, None]
    return c, s["k_pe"][p, r].double()


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "append":
        x, slots = s["kv_a"].double(), s["slots"]
        cos, sin = (s[k][s["positions"]].double() for k in ("cos", "sin"))
        n = x[:, :LATENT] / torch.sqrt((x[:, :LATENT] ** 2).sum(-1, keepdim=True) / LATENT + EPS) * s["weight"].double()
        k_pe = s["k_pe"].double()
        k_pe.view(-1, ROPE)[slots] = _turned(x[:, LATENT:], cos, sin)
        if s["scale"] is None:
            latent = s["latent"].double()
            latent.view(-1, LATENT)[slots] = n
            return {"latent": latent, "k_pe": k_pe, "scale": None}
        top = n.abs().max(-1).values / FP8_MAX
        scale, latent = s["scale"].double(), s["latent"].to(torch.float32).double()
        scale.view(-1)[slots] = top
        y = n / top[:, None]  # to the nearest of e4m3: steps of an eighth of the power of two below, no finer than 2^-9, ties to even
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
        latent.view(-1, LATENT)[slots] = torch.round(y / step) * step
        return {"latent": latent, "k_pe": k_pe, "scale": scale}
    if kind == "absorb":
        h = (s["o_latent"] if s["side"] == "value" else s["q"]).shape[1]
        w = s["weight"].double().reshape(h, NOPE + VALUE, LATENT)
        if s["side"] == "value":
            return torch.stack([s["o_latent"][:, i].double() @ w[i, NOPE:].T for i in range(h)], 1)
        q = s["q"].double()
        cos, sin = (s[k][s["positions"]].double()[:, None].expand(-1, h, -1) for k in ("cos", "sin"))
        return torch.stack([q[:, i, :NOPE] @ w[i, :NOPE] for i in range(h)], 1), _turned(q[..., NOPE:], cos, sin)
    lengths = _lengths(case)
    if kind == "gather":
        rows = [_exact_rows(s, i, length) for i, length in enumerate(lengths)]
        return torch.cat([c for c, _ in rows]), torch.cat([p for _, p in rows])
    outs, lses, first = [], [], 0
    for i, (n, length) in enumerate(zip(_counts(case), lengths)):
        c, p = _exact_rows(s, i, length)
        q = s["q_latent"][first : first + n].double(), s["q_pe"][first : first + n].double()
        score = (q[0] @ c.T + q[1] @ p.T) * (SCALE * math.log2(math.e))  # [n, h, length], in bits
        words = [(1 << t + 1) - 1 for t in range(n)] if s["tree"] is None else s["tree"][first : first + n].tolist()
        hidden = torch.tensor([[not w >> d & 1 for d in range(n)] for w in words], device="cuda")
        score[..., length - n :].masked_fill_(hidden[:, None], -math.inf)
        lse = torch.logsumexp(score * math.log(2.0), -1) / math.log(2.0)
        outs.append(torch.exp2(score - lse[..., None]) @ c)
        lses.append(lse.T)
        first += n
    return torch.cat(outs), torch.cat(lses, 1)
