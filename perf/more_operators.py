"""The operators of the key-value cache of the GQA layer as data and functions: what a serving or sampling loop of that layer runs.

  plan       the step's bookkeeping on the device: pages of requests that ended go back to a pool, pages for new rows come out of it; token offsets,
             positions and slots of the step (for this cache and the latent one alike)
  append     q and k per-head RMSNorm and rotation, k and v into cache pages (bf16, or e4m3 with a scale a row and head)
  attention  one or a few new tokens a sequence against its cached rows, causal
  tree       the same for a tree of drafted tokens, whose mask is a word of bits a token
  select     bounds of the pages that the step filled, then for every token and key-value head the pages whose bounds promise the highest scores
  sparse     attention of single tokens to the pages that were selected for them

`own` says who computes: False the plain form below, elementary torch operations in 32 bits (scores of pages, which decide a choice, in 64), True the framework's
operators. Heads are those of Qwen3-30B-A3B's layer (32 query and 4 key-value heads of 128), or generic ones. Imported with the root of the tree under
measurement as the working folder.
"""

import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
POSITIONS = 16384  # of the rotary tables


def _package():
    package = os.path.join(os.getcwd(), "pith-train_amd")
    if package not in sys.path:
        sys.path.insert(0, package)


def _cache_operators():
    _package()
    from pithtrain_amd.operators.gqa import kv_cache

    return kv_cache


def _paging_operators():
    _package()
    from pithtrain_amd.operators import paging

    return paging


# ---------------------------------------------------------------------------------------------
# Cases


def _plan(name, b, longest, new, page, spare=1.5):
    """b requests of up to `longest` cached rows and `new` new ones on average; spare: pages in the pool by those that are needed."""
    return {"name": name, "kind": "plan", "b": b, "longest": longest, "new": new, "page": page, "spare": spare}


def _append(name, tokens, run, cache, page, heads=(32, 4, 128), weight="bf16"):
    """`run` consecutive tokens a sequence: 1 while answering, the prompt's length while reading it. weight: of the norms, or "none"."""
    h, hkv, d = heads
    return {"name": name, "kind": "append", "tokens": tokens, "run": run, "cache": cache, "page": page, "h": h, "hkv": hkv, "d": d, "weight": weight}


def _attention(name, kind, b, q, longest, least, cache, page, heads=(32, 4, 128), even=True):
    """`q` new tokens a sequence (even) or 1 .. q; cached lengths, new tokens included, from least * longest to longest."""
    h, hkv, d = heads
    return {"name": name, "kind": kind, "b": b, "q": q, "longest": longest, "least": least, "cache": cache, "page": page, "h": h, "hkv": hkv, "d": d, "even": even}


def _pages_case(name, kind, b, q, longest, least, keep, cache, page, heads=(32, 4, 128)):
    """select and sparse: `keep` pages for every token and key-value head."""
    return dict(_attention(name, kind, b, q, longest, least, cache, page, heads), keep=keep)


def listed():
    return [
        # One step of 32 requests that are being answered: a row each, now and then a page. The smallest.
        _plan("plan_step", 32, 8192, 1, 64),
        # Prompts of 16 requests are read in, 16384 tokens in all; the pool does not suffice for the last ones.
        _plan("plan_prompts_scarce", 16, 4096, 1024, 16, spare=0.8),
        # The new rows of one step of 32 sequences go into 32 pages, quantised.
        _append("append_step_fp8", 32, 1, "fp8", 64),
        # A prompt of 8192 tokens is read in: the cache as bf16.
        _append("append_prompt", 8192, 8192, "bf16", 64),
        # The smallest attention: one sequence of a few hundred tokens.
        _attention("decode_small", "attention", 1, 1, 517, 1.0, "bf16", 64),
        # An ordinary step: 32 sequences of very different lengths.
        _attention("decode_batch", "attention", 32, 1, 8192, 0.1, "bf16", 64),
        # Long contexts from an fp8 cache: the largest by bytes.
        _attention("decode_long_fp8", "attention", 8, 1, 131072, 0.5, "fp8", 64),
        # Drafted tokens of a small model with heads of 64, trees of different sizes, small pages.
        _attention("tree_head64", "tree", 12, 8, 5001, 0.25, "bf16", 16, (16, 2, 64), even=False),
        # Which pages the 32 tokens of an ordinary step attend to.
        _pages_case("select_batch", "select", 32, 1, 8192, 0.1, 16, "bf16", 64),
        # The same for long contexts from an fp8 cache.
        _pages_case("select_long_fp8", "select", 8, 1, 131072, 0.5, 64, "fp8", 64),
        # Attention to 16 pages of each of 32 sequences.
        _pages_case("sparse_batch", "sparse", 32, 1, 8192, 0.1, 16, "bf16", 64),
        # Attention to 64 pages of each long context.
        _pages_case("sparse_long_fp8", "sparse", 8, 1, 131072, 0.5, 64, "fp8", 64),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


HEADS = [(32, 4, 128), (32, 4, 128), (32, 8, 128), (16, 2, 64), (64, 4, 128), (28, 4, 128), (8, 8, 64), (6, 2, 128), (5, 1, 64), (16, 1, 128)]


def _draw_any(rng):
    kind = rng.choice(["plan", "append", "attention", "attention", "attention", "tree", "select", "select", "sparse", "sparse"])
    cache, page, heads = rng.choice(["bf16", "fp8"]), rng.choice([16, 32, 64, 64, 128]), rng.choice(HEADS)
    least = rng.choice([0.05, 0.3, 0.7, 1.0])
    if kind == "plan":
        b = _log_int(rng, 1, 1024)
        new = rng.choice([1, _log_int(rng, 1, max(1, 65536 // b))])
        case = _plan("", b, _log_int(rng, 1, 32768), new, page, rng.choice([0.5, 0.9, 1.5, 1.5]))
    elif kind == "append":
        tokens = _log_int(rng, 1, 16384)
        run = rng.choice([1, tokens]) if tokens <= 256 else _log_int(rng, 64, tokens)
        case = _append("", tokens, run, cache, page, heads, rng.choice(["bf16", "bf16", "fp32", "none"]))
    elif kind in ("attention", "tree"):
        q = rng.choice([1, 1, 1, 2, 3, rng.randint(4, 16)]) if kind == "attention" else rng.randint(2, 24)
        case = _attention("", kind, _log_int(rng, 1, 128), q, _log_int(rng, 1, 131072), least, cache, page, heads, rng.random() < 0.5)
    else:
        q = rng.choice([1, 1, 1, 2, rng.randint(3, 8)]) if kind == "select" else 1
        case = _pages_case("", kind, _log_int(rng, 1, 128), q, _log_int(rng, 64, 131072), least, _log_int(rng, 2, 128), cache, page, heads)
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
        if case["kind"] == "plan" and case["b"] * case["longest"] > case["page"] << 18:  # lists that prepare makes on the host
            continue
        if "longest" in case and case["kind"] != "plan":  # what the plain form lays out: padded keys and scores in 32 bits
            rows = case["b"] * (case["keep"] * case["page"] if case["kind"] == "sparse" else max(_lengths(case)))
            if rows * case["hkv"] * case["d"] * 4 > 4 << 30 or rows * case["h"] * max(_counts(case)) * 4 > 4 << 30:
                continue
            if sum(_lengths(case)) * case["hkv"] * case["d"] > 1 << 29 or (case["kind"] == "select" and case["b"] * case["q"] > 512):  # what prepare lays out
                continue
        return case


def _counts(case):
    """New tokens of each sequence."""
    b, q = case["b"], case["q"]
    return [q if case["even"] else 1 + (7 * i + q - 1) % q for i in range(b)]


def _lengths(case):
    """Cached rows of each sequence, its new tokens among them: spread evenly between the shortest and the longest. With selection every fourth sequence fills a page."""
    spread = [(i * 0.6180339887498949) % 1.0 for i in range(case["b"])]
    least, longest = case["least"], case["longest"]
    lengths = [max(n, 1, int(round(longest * (1.0 - (1.0 - least) * f)))) for n, f in zip(_counts(case), spread)]
    if case["kind"] == "select":
        lengths = [-(-n // case["page"]) * case["page"] if i % 4 == 0 else n for i, n in enumerate(lengths)]
    return lengths


def _element(case):
    return 2 if case["cache"] == "bf16" else 1


def _row_bytes(case):
    """A key and a value of one head."""
    return 2 * (case["d"] * _element(case) + (4 if case["cache"] == "fp8" else 0))


def work(case):
    kind = case["kind"]
    if kind == "plan":
        b, tokens = case["b"], case["b"] * case["new"]
        return {"bytes": 4 * (6 * b + 3) + 16 * tokens + 8 * (tokens // case["page"] + b // 16), "flops": 0}
    h, hkv, d = case["h"], case["hkv"], case["d"]
    if kind == "append":
        t = case["tokens"]
        return {"bytes": t * (2 * d * (2 * h + 2 * hkv) + hkv * _row_bytes(case) + 4 * d + 16), "flops": t * (h + hkv) * 7 * d}
    counts, lengths = _counts(case), _lengths(case)
    t = sum(counts)
    if kind == "select":
        pages = [-(-n // case["page"]) for n in lengths]
        filled = sum(1 for n, length in zip(counts, lengths) for i in range(n) if (length - n + i + 1) % case["page"] == 0)
        scored = hkv * sum(n * p for n, p in zip(counts, pages))
        return {"bytes": hkv * sum(pages) * 4 * d + 2 * t * h * d + t * hkv * 4 * (case["keep"] + 1) + hkv * filled * (case["page"] * _row_bytes(case) // 2 + 4 * d),
                "flops": 4 * (h // hkv) * scored * d}  # fmt: skip
    if kind == "sparse":
        rows = [_kept_rows(case, length) for length in lengths]
        return {"bytes": hkv * sum(rows) * _row_bytes(case) + t * h * (4 * d + 4), "flops": 4 * h * sum(rows) * d}
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(counts, lengths))
    return {"bytes": hkv * sum(lengths) * _row_bytes(case) + t * h * (4 * d + 4), "flops": 4 * h * pairs * d}


def _kept_rows(case, length):
    """Rows of the pages that are kept of a sequence: its last page, which may be filled in part, and whole ones."""
    pages = -(-length // case["page"])
    return length - max(pages - case["keep"], 0) * case["page"]


# ---------------------------------------------------------------------------------------------
# What the program has in hand


def _tables(d, dev):
    angle = torch.arange(POSITIONS, device=dev, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
    angle = torch.cat((angle, angle), 1)
    return angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)


def _rows(case, pages, g, dev, std):
    """Pages [pages, heads, page, d] of keys or values: features of different size, with scales where the cache is e4m3."""
    hkv, d, page = case["hkv"], case["d"], case["page"]
    x = torch.randn(pages, hkv, page, d, generator=g, device=dev)
    x *= std * (0.5 + torch.rand(hkv, 1, d, generator=g, device=dev))
    if case["cache"] == "bf16":
        return x.to(torch.bfloat16), None
    scale = x.abs().amax(-1) / FP8_MAX
    x /= scale[..., None]
    return x.clamp_(-FP8_MAX, FP8_MAX).to(FP8), scale


def _cache(case, pages, g, dev, state):
    state["k"], state["k_scale"] = _rows(case, pages, g, dev, 1.0)
    state["v"], state["v_scale"] = _rows(case, pages, g, dev, 0.7)


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


def _prepare_plan(case, seed, dev):
    rng = random.Random(seed)
    b, page, tokens = case["b"], case["page"], case["b"] * case["new"]
    lengths = [rng.randint(0, case["longest"]) for _ in range(b)]
    most = 1 if case["new"] == 1 else 2 * case["new"]
    counts, left = [], tokens
    for _ in range(b):
        counts.append(min(left, 1 if most == 1 else rng.randint(0, most)))
        left -= counts[-1]
    for i in range(b):
        counts[i] = rng.choice([-1, 0]) if rng.random() < 0.1 else counts[i]  # ended, or waiting
    held = [-(-n // page) for n in lengths]
    need = sum(-(-(n + max(c, 0)) // page) - p for n, c, p in zip(lengths, counts, held))
    ended = sum(p for c, p in zip(counts, held) if c < 0)
    width = -(-(case["longest"] + most) // page) + 1
    order = list(range(b * width))
    rng.shuffle(order)
    table, at = [], 0
    for p in held:
        table.append(order[at : at + p] + [-1] * (width - p))
        at += p
    spare = min(max(int(case["spare"] * need) - ended, 0) + (1 if case["spare"] > 1 else 0), len(order) - at)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    free = order[at : at + spare] + [-1] * (len(order) - spare)  # the other pages belong to somebody else
    return {"kind": "plan", "tokens": tokens, "page": page, "counts": i32(counts), "lengths": i32(lengths), "page_table": i32(table), "free": i32(free), "count": i32([spare])}


def prepare(case, seed):
    dev = torch.device("cuda")
    kind = case["kind"]
    if kind == "plan":
        return _prepare_plan(case, seed, dev)
    g = torch.Generator(device=dev).manual_seed(seed)
    h, hkv, d, page = case["h"], case["hkv"], case["d"], case["page"]
    bf16 = lambda *s, std=1.0: (std * torch.randn(*s, generator=g, device=dev)).to(torch.bfloat16)  # noqa: E731
    state = {"kind": kind, "hkv": hkv, "page": page, "scale": d**-0.5}
    if kind == "append":
        t, run = case["tokens"], case["run"]
        runs = -(-t // run)
        per_run = -(-run // page)
        pages = runs * per_run + 2
        order = torch.randperm(pages, generator=g, device=dev)[: runs * per_run].view(runs, per_run)
        i = torch.arange(t, device=dev)
        at = i % run if run > 1 else torch.randint(0, page, (t,), generator=g, device=dev)
        _cache(case, pages, g, dev, state)
        state["slots"] = order[i // run, at // page] * page + at % page
        state["positions"] = at % POSITIONS if run > 1 else torch.randint(0, POSITIONS, (t,), generator=g, device=dev)
        qkv = bf16(t, (h + 2 * hkv) * d, std=1.5)  # one projection, as the program splits it
        state["q"], state["k_new"], state["v_new"] = (x.view(t, -1, d) for x in qkv.split((h * d, hkv * d, hkv * d), 1))
        dtype = torch.float32 if case["weight"] == "fp32" else torch.bfloat16
        for name in ("q_weight", "k_weight"):
            state[name] = None if case["weight"] == "none" else (1.0 + 0.2 * torch.randn(d, generator=g, device=dev)).to(dtype)
        state["cos"], state["sin"] = _tables(d, dev)
        return state
    lengths, counts = _lengths(case), _counts(case)
    t = sum(counts)
    state["q"] = bf16(t, h, d)
    table, pages = _page_table(case, lengths, g, dev)
    if kind == "select":
        state["keep"], state["most"] = case["keep"], max(counts)
        state["page_table"], state["lengths"], state["cu_q"] = table, torch.tensor(lengths, dtype=torch.int32, device=dev), _offsets(counts, dev)
        state["k"], state["k_scale"] = _rows(case, pages, g, dev, 1.0)
        state["v"], state["v_scale"] = state["k"], state["k_scale"]  # not looked at
        x = state["k"].float() if state["k_scale"] is None else state["k"].float() * state["k_scale"][..., None]
        state["bounds"] = torch.stack((x.amin(2), x.amax(2)), 2).to(torch.bfloat16)  # [pages, heads, 2, d]
        del x
        for i, (n, length) in enumerate(zip(counts, lengths)):  # those that this step fills are still to come
            for at in range(length - n, length):
                if (at + 1) % page == 0:
                    state["bounds"][table[i, at // page].long()] = 0.0
        return state
    _cache(case, pages, g, dev, state)
    if kind == "sparse":
        # for every head the pages that were selected, in their order, the sequence's last one among them
        b, keep = case["b"], case["keep"]
        need = torch.tensor([-(-n // page) for n in lengths], device=dev)
        rank = torch.rand(b, hkv, table.shape[1], generator=g, device=dev)
        j = torch.arange(table.shape[1], device=dev)
        rank = torch.where(j < need[:, None, None] - 1, rank, torch.where(j == need[:, None, None] - 1, 2.0, -1.0))
        rank = torch.cat((rank, torch.full((b, hkv, max(keep - table.shape[1], 0)), -1.0, device=dev)), 2)
        best = rank.topk(keep, -1)
        chosen = torch.where(best.values >= 0, best.indices, 1 << 30).sort(-1).values
        physical = table.long()[:, None].expand(-1, hkv, -1).gather(2, chosen.clamp(max=table.shape[1] - 1))
        state["page_table"] = torch.where(chosen < 1 << 30, physical, -1).to(torch.int32).contiguous()
        rows = [_kept_rows(case, n) for n in lengths]
        state["lengths"] = torch.tensor(rows, dtype=torch.int32, device=dev)[:, None].expand(b, hkv).contiguous()
        state["cu_q"], state["tree"], state["most"] = None, None, 1
        return state
    state["page_table"] = table
    state["most"] = max(counts)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
    state["cu_q"] = _offsets(counts, dev)
    state["tree"] = torch.tensor(_tree_words(case, seed), dtype=torch.int64, device=dev) if kind == "tree" else None
    return state


# ---------------------------------------------------------------------------------------------
# The plain form


def _plain_plan(s):
    page, tokens = s["page"], s["tokens"]
    table, free = s["page_table"], s["free"]
    b, width = table.shape
    lengths, counts = s["lengths"].long(), s["counts"].long()
    ended = counts < 0
    held = (lengths + page - 1) // page
    # pages of requests that ended, behind those that the pool holds
    j = torch.arange(width, device="cuda")
    back = (ended[:, None] & (j < held[:, None])).view(-1)
    order = torch.cumsum(back, 0) - 1 + s["count"].long()
    longer = torch.cat((free, free.new_zeros(1)))  # one more place for the entries that stay
    longer[torch.where(back, order, free.numel())] = table.view(-1)
    free[:] = longer[:-1]
    count = s["count"].long() + back.sum()
    # new rows: all of a request or none, in the order of the requests, until the pages do not suffice
    cu = torch.cat((torch.zeros(1, dtype=torch.long, device="cuda"), torch.cumsum(counts.clamp(min=0), 0))).clamp(max=tokens)
    new = cu[1:] - cu[:-1]
    after = lengths + new
    fits = ~ended & (after <= width * page)
    need = torch.where(fits, (after + page - 1) // page - held, 0)
    upto = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (upto <= count))
    rest = count - torch.where(granted, need, 0).sum()
    # rows of the tokens
    t = torch.arange(tokens, device="cuda")
    seq = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=b - 1)
    real = t < cu[-1]
    position = lengths[seq] + t - cu[seq]
    index = position // page
    taken = (count - 1 - (upto - need)[seq] - (index - held[seq])).clamp(0, free.numel() - 1)
    own_page = torch.where(index < held[seq], table.view(-1)[seq * width + index.clamp(max=width - 1)].long(), free[taken].long())
    has = real & granted[seq]
    slots = torch.where(has, own_page * page + position % page, -1)
    first = has & (index >= held[seq])
    longer = torch.cat((table.view(-1), table.new_zeros(1)))
    longer[torch.where(first, seq * width + index, b * width)] = own_page.to(torch.int32)
    table.view(-1)[:] = longer[:-1]
    i32 = torch.int32
    return {"cu_q": cu.to(i32), "positions": torch.where(real, position, 0), "slots": slots, "granted": torch.where(granted, new, 0).to(i32),
            "lengths": torch.where(ended, 0, torch.where(granted, after, lengths)).to(i32), "count": rest.to(i32).view(1), "page_table": table, "free": free}  # fmt: skip


def _normed(x, weight):
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _rotated(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat((-x[..., half:], x[..., :half]), -1) * sin


def _plain_append(s):
    cos, sin = s["cos"][s["positions"]].float()[:, None], s["sin"][s["positions"]].float()[:, None]
    q = _rotated(_normed(s["q"].float(), s["q_weight"]), cos, sin).to(torch.bfloat16)
    k = _rotated(_normed(s["k_new"].float(), s["k_weight"]), cos, sin)
    at, row = s["slots"] // s["page"], s["slots"] % s["page"]
    for name, x in (("k", k), ("v", s["v_new"].float())):
        if s["k_scale"] is None:
            s[name][at, :, row] = x.to(torch.bfloat16)
            continue
        scale = x.abs().amax(-1) / FP8_MAX
        s[name + "_scale"][at, :, row] = scale
        x = (x / scale[..., None]).clamp(-FP8_MAX, FP8_MAX).to(FP8)
        s[name].view(torch.uint8)[at, :, row] = x.view(torch.uint8)
    return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _pages(s, name):
    """Rows of the tables' pages, [b, heads, most rows, features] in 32 bits; a table is of all heads or of one each."""
    table = s["page_table"].long().clamp(min=0)
    if table.dim() == 2:
        table = table[:, None].expand(-1, s["hkv"], -1)
    head = torch.arange(s["hkv"], device="cuda")[None, :, None]
    x = s[name].view(torch.uint8)[table, head].view(s[name].dtype).float()
    if s[name + "_scale"] is not None:
        x *= s[name + "_scale"][table, head][..., None]
    return x.flatten(2, 3)


def _plain_attention(s):
    keys = _pages(s, "k")
    t, h, d = s["q"].shape
    b, hkv, n_keys, _ = keys.shape
    most, group = s["most"], h // hkv
    cu_q = torch.arange(b + 1, device="cuda") if s["cu_q"] is None else s["cu_q"].long()
    counts = cu_q[1:] - cu_q[:-1]
    lengths = s["lengths"].long() if s["lengths"].dim() == 2 else s["lengths"].long()[:, None]  # [b, heads or 1]
    i = torch.arange(most, device="cuda")
    token = (cu_q[:-1, None] + i).clamp(max=t - 1)  # [b, most]; what lies behind a sequence's own tokens is left out below
    q = s["q"].float()[token].view(b, most, hkv, group, d).transpose(1, 2).reshape(b, hkv, most * group, d)
    score = torch.matmul(q, keys.transpose(2, 3).contiguous()).mul_(s["scale"])
    del keys
    before = (lengths - counts[:, None])[..., None, None]  # keys in front of the new tokens, [b, heads or 1, 1, 1]
    j = torch.arange(n_keys, device="cuda")
    if s["tree"] is None:
        seen = j <= before + i[:, None]
    else:
        bit = (j - before).clamp(0, 63)
        seen = (j < before) | ((s["tree"][token][:, None, :, None] >> bit) & 1).bool()
    seen = seen & (j < lengths[..., None, None])
    score = score.view(b, hkv, most, group, n_keys).masked_fill_(~seen[:, :, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), _pages(s, "v")).view(b, hkv, most, group, d) / torch.where(total == 0, 1.0, total)
    lse = ((top + torch.log(total)) * (1.0 / math.log(2.0)))[..., 0]
    o, lse = o.transpose(1, 2).reshape(b, most, h, d), lse.transpose(1, 2).reshape(b, most, h)
    every = torch.arange(t, device="cuda")
    seq = torch.searchsorted(cu_q, every, right=True) - 1
    mine = every - cu_q[seq]
    return o[seq, mine].to(torch.bfloat16), lse[seq, mine].t().contiguous()


def _plain_select(s):
    page, keep, hkv = s["page"], s["keep"], s["hkv"]
    table, cu_q, lengths = s["page_table"].long(), s["cu_q"].long(), s["lengths"].long()
    t, h, d = s["q"].shape
    every = torch.arange(t, device="cuda")
    seq = torch.searchsorted(cu_q, every, right=True) - 1
    visible = lengths[seq] - cu_q[seq + 1] + every + 1
    pages = (visible + page - 1) // page  # of each token, its own the last
    # bounds of the pages whose last row is a new one
    own_page = table[seq, pages - 1]
    x = s["k"].view(torch.uint8)[own_page].view(s["k"].dtype).float()
    if s["k_scale"] is not None:
        x = x * s["k_scale"][own_page][..., None]
    x = torch.stack((x.amin(2), x.amax(2)), 2).to(torch.bfloat16)
    filled = visible % page == 0
    longer = torch.cat((s["bounds"], s["bounds"][:1]))
    longer[torch.where(filled, own_page, len(s["bounds"]))] = x
    s["bounds"][:] = longer[:-1]
    # scores: a bound of q . k over a page, the largest of the heads that share it
    width = table.shape[1]
    q = s["q"].double().view(t, hkv, h // hkv, d)
    signs = torch.cat((q.clamp(max=0), q.clamp(min=0)), -1)  # against (lowest, highest)
    of_seq = s["bounds"][table].transpose(1, 2).flatten(3)  # [b, heads, pages, 2 d]
    score = torch.empty(t, hkv, width, device="cuda")
    for i0 in range(0, t, 8):
        part = of_seq[seq[i0 : i0 + 8]].double()
        score[i0 : i0 + 8] = torch.matmul(signs[i0 : i0 + 8], part.transpose(2, 3)).amax(2).float()
    j = torch.arange(width, device="cuda")
    score = torch.where(j < (pages - 1)[:, None, None], score + 0.0, -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., : keep - 1]
    best = torch.cat((best, best.new_full((t, hkv, keep - 1 - best.shape[-1]), 1 << 30)), -1)
    rank = torch.arange(keep - 1, device="cuda")
    best = torch.where(rank < (pages - 1)[:, None, None], best, 1 << 30).sort(-1).values
    n = torch.clamp(pages, max=keep)  # pages of each token that are kept
    best = torch.cat((best, best.new_full((t, hkv, 1), 1 << 30)), -1)
    best = torch.where(torch.arange(keep, device="cuda") == (n - 1)[:, None, None], (pages - 1)[:, None, None], best)
    physical = table[seq][:, None].expand(-1, hkv, -1).gather(2, best.clamp(max=width - 1))
    chosen = torch.where(best < 1 << 30, physical, -1).to(torch.int32)
    rows = (visible - (pages - n) * page).to(torch.int32)
    return {"bounds": s["bounds"], "page_table": chosen, "lengths": rows[:, None].expand(-1, hkv).contiguous()}


def run(state):
    s = state
    kind = s["kind"]
    if not own:
        if kind == "plan":
            return _plain_plan(s)
        if kind == "append":
            return _plain_append(s)
        return _plain_select(s) if kind == "select" else _plain_attention(s)
    if kind == "plan":
        ops = _paging_operators()
        plan = ops.plan_step(s["counts"], s["lengths"], s["page_table"], ops.PagePool(s["free"], s["count"]), s["page"], s["tokens"])
        return {"cu_q": plan.cu_q, "positions": plan.position_ids, "slots": plan.slots, "granted": plan.granted, "lengths": plan.lengths,
                "count": plan.free_count, "page_table": s["page_table"], "free": s["free"]}  # fmt: skip
    ops = _cache_operators()
    cache = ops.KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if kind == "append":
        q = ops.kv_cache_append(s["q"], s["k_new"], s["v_new"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"], s["slots"], cache, EPS)
        return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if kind == "select":
        ops.kv_page_bounds(cache, s["bounds"], s["page_table"], s["lengths"], s["cu_q"], s["q"].shape[0])
        chosen = ops.kv_select_pages(s["q"], s["bounds"], s["page_table"], s["lengths"], s["cu_q"], s["page"], s["keep"])
        return {"bounds": s["bounds"], "page_table": chosen.page_table, "lengths": chosen.lengths}
    return ops.kv_attention(s["q"], cache, s["page_table"], s["lengths"], s["cu_q"], s["scale"], s["tree"])


# ---------------------------------------------------------------------------------------------
# The definition in 64 bits


def _exact_plan(s):
    page, tokens = s["page"], s["tokens"]
    counts, lengths, table = s["counts"].tolist(), s["lengths"].tolist(), s["page_table"].tolist()
    free, count = s["free"].tolist(), int(s["count"])
    for i, n in enumerate(counts):
        if n < 0:
            for p in table[i][: -(-lengths[i] // page)]:
                free[count] = p
                count += 1
            lengths[i] = 0
    cu, positions, slots, granted, short, top = [0], [], [], [], False, count
    for i, n in enumerate(counts):
        n = max(n, 0)
        held = -(-lengths[i] // page)
        need = -(-(lengths[i] + n) // page) - held
        takes = counts[i] >= 0 and (need == 0 or (not short and need <= top))
        short = short or (counts[i] >= 0 and not takes)
        for j in range(need if takes else 0):
            top -= 1
            table[i][held + j] = free[top]
        for k in range(n):
            at = lengths[i] + k
            positions.append(at)
            slots.append(table[i][at // page] * page + at % page if takes else -1)
        granted.append(n if takes else 0)
        lengths[i] += granted[-1]
        cu.append(cu[-1] + n)
    positions += [0] * (tokens - len(positions))
    slots += [-1] * (tokens - len(slots))
    mk = lambda x, like: torch.tensor(x, dtype=like, device="cuda")  # noqa: E731
    i32, i64 = torch.int32, torch.int64
    return {"cu_q": mk(cu, i32), "positions": mk(positions, i64), "slots": mk(slots, i64), "granted": mk(granted, i32), "lengths": mk(lengths, i32),
            "count": mk([top], i32), "page_table": mk(table, i32), "free": mk(free, i32)}  # fmt: skip


def _turned(x, cos, sin):
    """The rotation as complex numbers: features (j, j + d / 2) are real and imaginary part, times cos_j + i sin_j."""
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * torch.complex(cos[..., :half].contiguous(), sin[..., :half].contiguous())
    return torch.cat((z.real, z.imag), -1)


def _exact_append(s):
    cos, sin = (s[k][s["positions"]].double()[:, None] for k in ("cos", "sin"))

    def normed(x, weight):
        x = x.double()
        return x if weight is None else x / torch.sqrt((x**2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()

    out = {"q": _turned(normed(s["q"], s["q_weight"]), *(c.expand(-1, s["q"].shape[1], -1) for c in (cos, sin)))}
    k = _turned(normed(s["k_new"], s["k_weight"]), *(c.expand(-1, s["hkv"], -1) for c in (cos, sin)))
    page, row = torch.div(s["slots"], s["page"], rounding_mode="floor"), s["slots"] % s["page"]
    for name, x in (("k", k), ("v", s["v_new"].double())):
        rows, scales = s[name].to(torch.float32).double(), None
        if s["k_scale"] is not None:
            top = x.abs().max(-1).values / FP8_MAX
            scales = s[name + "_scale"].double()
            scales[page, :, row] = top
            y = x / top[..., None]  # to the nearest of e4m3: steps of an eighth of the power of two below, no finer than 2^-9, ties to even
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
            x = torch.round(y / step) * step
        rows[page, :, row] = x
        out[name], out[name + "_scale"] = rows, scales
    return out


def _exact_rows(s, name, table, head, length):
    """Rows 0 .. length - 1 of one table row and head."""
    at = torch.arange(length, device="cuda")
    p, r = table[at // s["page"]].long(), at % s["page"]
    x = s[name].view(torch.uint8)[p, head, r].view(s[name].dtype).double()
    return x if s[name + "_scale"] is None else x * s[name + "_scale"][p, head, r].double()[:, None]


def _exact_attention(s):
    t, h, d = s["q"].shape
    group = h // s["hkv"]
    b = len(s["page_table"])
    cu = list(range(b + 1)) if s["cu_q"] is None else s["cu_q"].tolist()
    lengths = s["lengths"].tolist()
    o, lse = torch.empty(t, h, d, dtype=torch.double, device="cuda"), torch.empty(h, t, dtype=torch.double, device="cuda")
    for i in range(b):
        first, n = cu[i], cu[i + 1] - cu[i]
        words = [(1 << k + 1) - 1 for k in range(n)] if s["tree"] is None else s["tree"][first : first + n].tolist()
        hidden = torch.tensor([[not w >> k & 1 for k in range(n)] for w in words], device="cuda")
        for head in range(s["hkv"]):
            table, length = (s["page_table"][i], lengths[i]) if s["page_table"].dim() == 2 else (s["page_table"][i, head], lengths[i][head])
            k, v = (_exact_rows(s, name, table, head, length) for name in ("k", "v"))
            mine = slice(head * group, (head + 1) * group)
            score = s["q"][first : first + n, mine].double() @ k.T * (s["scale"] * math.log2(math.e))  # [n, group, length], in bits
            score[..., length - n :].masked_fill_(hidden[:, None], -math.inf)
            total = torch.logsumexp(score * math.log(2.0), -1) / math.log(2.0)
            o[first : first + n, mine] = torch.exp2(score - total[..., None]) @ v
            lse[mine, first : first + n] = total.T
    return o, lse


def _exact_select(s):
    page, keep, hkv = s["page"], s["keep"], s["hkv"]
    t, h, _ = s["q"].shape
    cu, lengths = s["cu_q"].tolist(), s["lengths"].tolist()
    bounds, stored = s["bounds"].double(), s["bounds"].clone()
    chosen, rows = torch.full((t, hkv, keep), -1, dtype=torch.int32, device="cuda"), torch.empty(t, hkv, dtype=torch.int32, device="cuda")
    for i, length in enumerate(lengths):
        n = cu[i + 1] - cu[i]
        for full in range((length - n) // page, length // page):  # pages that are full now and were not before
            p = s["page_table"][i, full].long()
            x = s["k"][p].float().double()
            if s["k_scale"] is not None:
                x = x * s["k_scale"][p].double()[..., None]
            bounds[p, :, 0], bounds[p, :, 1] = x.min(1).values, x.max(1).values
            stored[p] = bounds[p].to(torch.bfloat16)
    for i, length in enumerate(lengths):
        mine = stored[s["page_table"][i].long()].double()  # [pages, heads, 2, d]
        for token in range(cu[i], cu[i + 1]):
            visible = length - cu[i + 1] + token + 1
            pages = -(-visible // page)
            q = s["q"][token].double().view(1, hkv, h // hkv, -1)
            best = torch.arange(pages - 1, device="cuda")[None].expand(hkv, -1)
            if pages > keep:
                score = torch.maximum(q * mine[: pages - 1, :, :1], q * mine[: pages - 1, :, 1:]).sum(-1).max(-1).values
                score = score.float().T.cpu().tolist()  # as the operator defines it: rounded once, equal ones by their page
                best = torch.tensor([sorted(sorted(range(pages - 1), key=lambda j: (-row[j], j))[: keep - 1]) for row in score], dtype=torch.long, device="cuda")
            best = best.reshape(hkv, min(pages, keep) - 1)
            chosen[token, :, : best.shape[1]] = s["page_table"][i][best]
            chosen[token, :, best.shape[1]] = s["page_table"][i, pages - 1]
            rows[token] = visible - max(pages - keep, 0) * page
    return {"bounds": bounds, "page_table": chosen, "lengths": rows}


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "plan":
        return _exact_plan(s)
    if kind == "append":
        return _exact_append(s)
    return _exact_select(s) if kind == "select" else _exact_attention(s)
