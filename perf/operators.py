"""The serving operators of drafted decoding over a shared prompt, as a benchmark: their cases, inputs and plain forms.

Three operators are run, each on its own:

  cache   new key and value rows are quantised into a paged 8-bit cache as they are appended (one f32 scale for each
          row of a head), and the same rows are read back at the values they stand for
  attend  the queries of a batch attend to one prefix that every sequence shares (a tool list, a system prompt) and to
          the sequence's own tail, causally, over that cache
  verify  drafted tokens are checked against the target's probabilities with given random numbers; the first rejected
          place is filled from what the target has above the draft, a run without rejection gets one more token

With `own` false, run() computes them in elementary torch operations; with `own` true it calls rustyneedle_b200.
"""

import math

import torch

own = False

PAGE = 64  # positions of a cache page
NONE = -1  # "no token" (UINT32_MAX of the C ABI, read as int32)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# Share of drafted tokens that prepare()'s drafts see accepted: about this at the noise used below. work() counts the
# target rows that a verification has to look at with it (those up to the first rejection).
KEPT = 0.75
NOISE = 0.7


# ---------------------------------------------------------------------------------------------------------- the cases


def listed():
    def cache(name, **k):
        return {"name": name, "op": "cache", "ragged": False, **k}

    def attend(name, **k):
        return {"name": name, "op": "attend", "ragged": False, **k}

    def verify(name, **k):
        return {"name": name, "op": "verify", "ragged": False, "given": True, "masked": False, "temperature": 1.0, **k}

    return [
        # one token of one sequence at this repository's geometry (4 heads of 64): nothing but latency
        cache("cache_one_token", sequences=1, rows=1, past=500, kv_heads=4, dim=64, format="int8", dtype="bf16"),
        # a decode step's rows: five for each of 256 sequences (four drafts and the token before them), pages half full
        cache("cache_draft_rows", sequences=256, rows=5, past=1000, kv_heads=4, dim=64, format="int8", dtype="fp16"),
        # a packed pass of ragged prompts, 40 to 1000 odd tokens each
        cache("cache_ragged_prompts", sequences=48, rows=1021, ragged=True, past=200, kv_heads=8, dim=128, format="e4m3", dtype="bf16"),
        # one user behind a 512-token prompt: this repository's batch-1 decoding
        attend("attend_one_user", sequences=1, rows=1, prefix=512, tail=77, heads=8, kv_heads=4, dim=64, format="int8", dtype="bf16"),
        # this repository's 256-sequence batch behind one tool list, tails up to 1000
        attend("attend_batch_256", sequences=256, rows=1, prefix=1000, tail=1000, heads=8, kv_heads=4, dim=64, format="int8", dtype="fp16"),
        # drafted tokens: 1 to 5 queries for each of 64 sequences over a long shared prompt
        attend("attend_drafts", sequences=64, rows=5, ragged=True, prefix=8200, tail=700, heads=32, kv_heads=8, dim=128, format="int8", dtype="bf16"),
        # a very long shared document, short answers: the largest
        attend("attend_long_document", sequences=128, rows=1, prefix=40000, tail=333, heads=32, kv_heads=8, dim=128, format="e4m3", dtype="bf16"),
        # the questions themselves being read behind the shared prompt: hundreds of queries each
        attend("attend_questions", sequences=6, rows=601, ragged=True, prefix=2500, tail=700, heads=16, kv_heads=4, dim=128, format="int8", dtype="fp16"),
        # four drafts of one sequence at this repository's vocabulary
        verify("verify_one_user", sequences=1, drafts=4, vocab=8192, dtype="fp32"),
        # the batch under grammar masks, ragged drafts
        verify("verify_masked_batch", sequences=256, drafts=4, ragged=True, vocab=8192, dtype="fp32", masked=True, temperature=0.8),
        # a large vocabulary of odd size, 16-bit logits
        verify("verify_large_vocabulary", sequences=96, drafts=5, vocab=129283, dtype="bf16"),
        # greedy verification of point drafts (an n-gram lookup): no draft probabilities
        verify("verify_greedy_lookup", sequences=200, drafts=7, vocab=50257, dtype="fp16", given=False, temperature=0.0),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["cache", "attend", "attend", "verify"])
    ragged = rng.random() < 0.6
    if op == "cache":
        case = {"op": op, "sequences": _log_uniform(rng, 1, 256), "rows": _log_uniform(rng, 1, 1100), "ragged": ragged,
                "past": rng.choice([0, 0, 1]) * _log_uniform(rng, 1, 1500), "kv_heads": rng.choice([1, 2, 3, 4, 8]), "dim": rng.choice([64, 128]),
                "format": rng.choice(["int8", "e4m3"]), "dtype": rng.choice(["bf16", "fp16", "fp32"])}
        while _cost(case) > 45e6 * 8:
            case["rows"] = case["rows"] // 2 + 1
            case["sequences"] = max(1, case["sequences"] - case["sequences"] // 4)
        return case
    if op == "attend":
        kv = rng.choice([1, 2, 4, 8])
        rows = _log_uniform(rng, 1, 700) if rng.random() < 0.3 else _log_uniform(rng, 1, 8)
        case = {"op": op, "sequences": _log_uniform(rng, 1, 256), "rows": rows, "ragged": ragged,
                "prefix": rng.choice([0, 1, 1, 1, 1]) * _log_uniform(rng, 1, 40000), "tail": max(rows, _log_uniform(rng, 1, 2000)),
                "heads": kv * rng.choice([1, 2, 3, 4, 5, 8]), "kv_heads": kv, "dim": rng.choice([64, 128]),
                "format": rng.choice(["int8", "e4m3"]), "dtype": rng.choice(["bf16", "fp16"])}
        while _cost(case) > 60e9:
            case["prefix"] = case["prefix"] * 3 // 4
            case["sequences"] = max(1, case["sequences"] - case["sequences"] // 8)
            case["rows"] = max(1, case["rows"] - case["rows"] // 8)
        return case
    greedy = rng.random() < 0.25
    case = {"op": op, "sequences": _log_uniform(rng, 1, 256), "drafts": rng.randint(1, 8), "ragged": ragged, "vocab": _log_uniform(rng, 500, 150000),
            "dtype": rng.choice(["fp32", "bf16", "fp16"]), "masked": rng.random() < 0.4, "given": rng.random() < 0.75,
            "temperature": 0.0 if greedy else rng.choice([1.0, 0.7, 1.3])}
    while _cost(case) > 75e6:
        case["sequences"] = max(1, case["sequences"] - case["sequences"] // 4)
        case["vocab"] = case["vocab"] * 7 // 8
    return case


def _cost(case):
    if case["op"] == "cache":
        return sum(_rows(case)) * case["kv_heads"] * case["dim"] * 8
    if case["op"] == "attend":
        return work(case)["flops"]
    return case["sequences"] * (case["drafts"] + 1) * case["vocab"]


def _spread(b, low, high):
    """A number of [low, high] for sequence b, spread evenly over the batch."""
    return low + int((b * 0.6180339887498949 + 0.35) % 1.0 * (high - low + 1))


def _rows(case):
    """New rows (queries) of each sequence; ragged batches of four and more have one sequence without any."""
    n, most = case["sequences"], case["rows"]
    if not case["ragged"]:
        return [most] * n
    rows = [_spread(b, max(1, most // 25), most) for b in range(n)]
    rows[0] = most
    if n >= 4:
        rows[2] = 0
    return rows


def _lengths(case):
    """Cached positions of each sequence behind its new rows, those included."""
    rows = _rows(case)
    if case["op"] == "cache":
        return [r + (_spread(3 * b + 1, 0, case["past"]) if case["past"] else 0) for b, r in enumerate(rows)]
    return [max(r, _spread(3 * b + 1, min(r, case["tail"]), case["tail"])) for b, r in enumerate(rows)]


def _drafted(case):
    n, k = case["sequences"], case["drafts"]
    return [_spread(b, 0, k) if case["ragged"] else k for b in range(n)]


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "cache":
        rows = sum(_rows(case)) * case["kv_heads"] * 2
        # rows in, codes and scales out and in again, values out
        return {"bytes": rows * (2 * case["dim"] * size + 2 * (case["dim"] + 4)), "flops": rows * case["dim"] * 3}
    if case["op"] == "attend":
        rows, lengths = _rows(case), _lengths(case)
        pairs = sum(r * case["prefix"] + r * (t - r) + r * (r + 1) // 2 for r, t in zip(rows, lengths))
        cached = case["prefix"] + sum(t for r, t in zip(rows, lengths) if r)
        return {"bytes": 2 * sum(rows) * case["heads"] * case["dim"] * size + 2 * cached * case["kv_heads"] * (case["dim"] + 4),
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    # the target's rows up to the first rejection (or the one behind the last draft), the draft's row at that place
    seen = sum(sum(KEPT**i for i in range(k + 1)) for k in _drafted(case))
    row = case["vocab"] * size + (case["vocab"] // 8 if case["masked"] else 0)
    drafts = case["sequences"] * case["vocab"] * 4 * (1 - KEPT) if case["given"] and case["temperature"] > 0 else 0
    return {"bytes": seen * row + drafts, "flops": seen * case["vocab"] * 4}


# --------------------------------------------------------------------------------------------------------- the inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(rows):
    at = [0]
    for r in rows:
        at.append(at[-1] + r)
    return at


def _fused_rows(g, rows, heads, kv_heads, dim, dtype):
    """Queries, keys and values as a fused projection leaves them: strided views of one buffer. Keys have a few strong
    channels, rows differ in size."""
    width = (heads + 2 * kv_heads) * dim
    x = torch.randn(rows, width, generator=g, device="cuda")
    channel = torch.exp(0.5 * torch.randn(width, generator=g, device="cuda"))
    x = (x * channel * torch.exp(0.3 * torch.randn(rows, 1, generator=g, device="cuda"))).to(dtype)
    cut = x.view(rows, heads + 2 * kv_heads, dim)
    return cut[:, :heads], cut[:, heads : heads + kv_heads], cut[:, heads + kv_heads :]


def _pages(g, lengths, before=0):
    """Page tables [sequences][most pages] in a shuffled pool, and the pool's number of pages (`before` pages are the prefix's)."""
    need = [-(-t // PAGE) for t in lengths]
    stride = max(1, max(need))
    total = before + sum(need)
    order = torch.randperm(max(1, total), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lengths), stride, dtype=torch.int32, device="cuda")
    at = before
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    return order[:before].contiguous(), table, max(1, total)


def _slots(rows, lengths):
    """For each new row its sequence and its position there."""
    sequence = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows))
    position = [torch.arange(t - r, t) for r, t in zip(rows, lengths)]
    return sequence.cuda(), (torch.cat(position) if position else torch.zeros(0, dtype=torch.long)).cuda()


def prepare(case, seed):
    return {"cache": _prepare_cache, "attend": _prepare_attend, "verify": _prepare_verify}[case["op"]](case, seed)


def _prepare_cache(case, seed):
    g = _generator(seed)
    rows, lengths = _rows(case), _lengths(case)
    kv, dim, dtype = case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    _, keys, values = _fused_rows(g, sum(rows), 2 * kv, kv, dim, dtype)
    _, table, total = _pages(g, lengths)
    s = {"case": case, "keys": keys, "values": values, "keys_out": torch.zeros(sum(rows), kv, dim, dtype=dtype, device="cuda"),
         "values_out": torch.zeros(sum(rows), kv, dim, dtype=dtype, device="cuda")}
    row_start, length = _int32(_starts(rows)), _int32(lengths)
    if own:
        import rustyneedle_b200 as nb

        s["cache"] = nb.KvCache(kv, dim, total, format=case["format"], device=0)
        s["batch"] = nb.KvBatch(row_start, length, table, rows=sum(rows), max_rows=max(rows), max_length=max(lengths))
    else:
        sequence, position = _slots(rows, lengths)
        s["page"], s["place"] = table[sequence, position // PAGE].long(), position % PAGE
        s["codes"] = torch.zeros(2, total, PAGE, kv, dim, dtype=torch.int8 if case["format"] == "int8" else torch.float8_e4m3fn, device="cuda")
        s["scales"] = torch.ones(2, total, PAGE, kv, device="cuda")
    return s


def _prepare_attend(case, seed):
    g = _generator(seed)
    rows, lengths, prefix = _rows(case), _lengths(case), case["prefix"]
    heads, kv, dim, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    query, _, _ = _fused_rows(g, sum(rows), heads, kv, dim, dtype)
    query *= 0.6
    _, keys, values = _fused_rows(g, prefix + sum(lengths), 0, kv, dim, dtype)
    prefix_pages, table, total = _pages(g, lengths, -(-prefix // PAGE))
    s = {"case": case, "query": query, "out": torch.zeros(sum(rows), heads, dim, dtype=dtype, device="cuda"), "prefix_pages": prefix_pages, "table": table}
    row_start, length = _int32(_starts(rows)), _int32(lengths)
    if own:
        import rustyneedle_b200 as nb

        s["cache"] = nb.KvCache(kv, dim, total, format=case["format"], device=0)
        if prefix:
            s["cache"].append(nb.KvBatch(_int32([0, prefix]), _int32([prefix]), prefix_pages[None], rows=prefix, max_rows=prefix, max_length=prefix),
                              keys[:prefix], values[:prefix])
        whole = nb.KvBatch(_int32(_starts(lengths)), length, table, rows=sum(lengths), max_rows=max(lengths), max_length=max(lengths))
        s["cache"].append(whole, keys[prefix:], values[prefix:])
        s["batch"] = nb.KvBatch(row_start, length, table, rows=sum(rows), max_rows=max(rows), max_length=max(lengths))
    else:
        sequence, position = _slots(lengths, lengths)
        page = torch.cat([prefix_pages[torch.arange(prefix, device="cuda") // PAGE], table[sequence, position // PAGE]]).long()
        place = torch.cat([torch.arange(prefix, device="cuda"), position]) % PAGE
        codes, scales = _quantise(torch.stack([keys, values]), case["format"])
        s["codes"] = torch.zeros(2, total, PAGE, kv, dim, dtype=codes.dtype, device="cuda")
        s["scales"] = torch.ones(2, total, PAGE, kv, device="cuda")
        if codes.dtype == torch.int8:
            s["codes"][:, page, place] = codes
        else:
            s["codes"].view(torch.int8)[:, page, place] = codes.view(torch.int8)
        s["scales"][:, page, place] = scales
        most = max(rows)
        of, at = torch.tensor(rows)[:, None], torch.arange(most)[None]
        s["row"] = torch.minimum(torch.tensor(_starts(rows)[:-1])[:, None] + at, torch.tensor(max(0, sum(rows) - 1))).cuda()
        s["live"] = (at < of).cuda()
        # the last position that each query sees in its own tail
        s["sees"] = (torch.tensor(lengths)[:, None] - of + at).cuda()
    return s


def _prepare_verify(case, seed):
    g = _generator(seed)
    n, k, v = case["sequences"], case["drafts"], case["vocab"]
    counts = _drafted(case)
    exact = 2.0 * torch.randn(n, k + 1, v, generator=g, device="cuda")
    exact.sub_(torch.empty(n, k + 1, v, device="cuda").exponential_(1.0, generator=g).mul_(1.5))
    # one token of each place stands out, by more or by less
    exact.scatter_add_(2, torch.randint(v, (n, k + 1, 1), generator=g, device="cuda"), 4 + 14 * torch.rand(n, k + 1, 1, generator=g, device="cuda"))
    logits = exact.to(DTYPES[case["dtype"]], copy=True)
    mask = None
    allowed = torch.ones(1, 1, 1, dtype=torch.bool, device="cuda")
    if case["masked"]:
        allowed = torch.rand(n, k + 1, v, generator=g, device="cuda") < 0.2
        allowed[:, 1] = allowed[:, 1] & (torch.rand(n, 1, generator=g, device="cuda") < 0.9)  # some states allow nothing
        allowed[:, 0, 7] = True
        mask = _pack(allowed)
    exact.add_(torch.randn(n, k + 1, v, generator=g, device="cuda"), alpha=NOISE)
    some = allowed.any(-1, keepdim=True)
    exact.masked_fill_(~(allowed | ~some), -math.inf)
    exact = exact[:, :k]
    if case["temperature"] > 0:
        draft = torch.softmax(exact / case["temperature"], -1)
        tokens = torch.multinomial(draft.view(n * k, v), 1, generator=g).view(n, k)
        if not case["given"]:
            tokens = torch.where(torch.rand(n, k, generator=g, device="cuda") < 0.6, logits[:, :k].float().masked_fill(~(allowed | ~some)[:, :k], -math.inf).argmax(-1), tokens)
    else:
        draft = torch.softmax(exact, -1)
        tokens = exact.argmax(-1)
    return {"case": case, "logits": logits, "mask": mask, "draft": draft if case["given"] else None, "tokens": tokens.to(torch.int32),
            "counts": _int32(counts), "accept": torch.rand(n, k, generator=g, device="cuda"), "sample": torch.rand(n, generator=g, device="cuda")}


def _pack(allowed):
    n, r, v = allowed.shape
    words = -(-v // 32)
    bits = torch.zeros(n, r, words * 32, dtype=torch.int64, device="cuda")
    bits[..., :v] = allowed
    bits = (bits.view(n, r, words, 32) << torch.arange(32, device="cuda")).sum(-1)
    return torch.where(bits >= 2**31, bits - 2**32, bits).to(torch.int32)


# ------------------------------------------------------------------------------------------------------ the operators


def run(state):
    return {"cache": _run_cache, "attend": _run_attend, "verify": _run_verify}[state["case"]["op"]](state)


def _run_cache(s):
    if own:
        s["cache"].append(s["batch"], s["keys"], s["values"])
        s["cache"].read(s["batch"], s["keys_out"], s["values_out"])
        return s["keys_out"], s["values_out"]
    codes, scales = _quantise(torch.stack([s["keys"], s["values"]]), s["case"]["format"])
    if codes.dtype == torch.int8:
        s["codes"][:, s["page"], s["place"]] = codes
    else:
        s["codes"].view(torch.int8)[:, s["page"], s["place"]] = codes.view(torch.int8)
    s["scales"][:, s["page"], s["place"]] = scales
    back = _values(s["codes"], s["scales"], s["page"], s["place"]).to(s["keys"].dtype)
    return back[0], back[1]


def _quantise(x, kind):
    """Codes [..., dim] and scales [...] of rows x [..., dim]. int8: the row's peak is 127 steps. e4m3: the smallest power
    of two that brings the peak to 448 or below. An empty row has scale 1. Quotients are formed in 64 bits: a quotient next
    to the middle between two codes has to fall on its own side."""
    peak = x.abs().amax(-1).float()
    if kind == "int8":
        scale = torch.where(peak > 0, peak / 127.0, torch.ones_like(peak))
        return torch.round(x.double() / scale.double()[..., None]).to(torch.int8), scale
    part, exponent = torch.frexp(peak)
    exponent = exponent - 9 + (part > 0.875)
    scale = torch.where(peak > 0, torch.ldexp(torch.ones_like(peak), exponent), torch.ones_like(peak))
    return (x.float() / scale[..., None]).to(torch.float8_e4m3fn), scale


def _values(codes, scales, page, place):
    """The cached values at (page, place), in 32 bits."""
    if codes.dtype == torch.int8:
        return codes[:, page, place].float() * scales[:, page, place][..., None]
    return codes.view(torch.int8)[:, page, place].view(torch.float8_e4m3fn).float() * scales[:, page, place][..., None]


def _run_attend(s):
    if own:
        s["cache"].attend(s["batch"], s["query"], s["out"], s["prefix_pages"], s["case"]["prefix"])
        return s["out"]
    case = s["case"]
    n, most = s["row"].shape
    kv, dim, prefix = case["kv_heads"], case["dim"], case["prefix"]
    group = case["heads"] // kv
    at = torch.arange(prefix, device="cuda")
    shared = _values(s["codes"], s["scales"], s["prefix_pages"].long()[at // PAGE], at % PAGE)  # [2, prefix, kv, dim]
    own_at = torch.arange(s["table"].shape[1] * PAGE, device="cuda")
    tail = _values(s["codes"], s["scales"], s["table"].long()[:, own_at // PAGE], (own_at % PAGE)[None].expand(n, -1))  # [2, n, tail, kv, dim]
    q = s["query"][s["row"]].float() / math.sqrt(dim)  # [n, most, heads, dim]
    q = q.view(n, most, kv, group, dim).permute(2, 0, 1, 3, 4)  # [kv, n, most, group, dim]
    width = own_at.numel()
    far = (q.reshape(kv, n * most * group, dim) @ shared[0].permute(1, 2, 0)).view(kv, n, most, group, prefix)
    near = (q.reshape(kv, n, most * group, dim) @ tail[0].permute(2, 0, 3, 1)).view(kv, n, most, group, width)
    near = near.masked_fill(~(own_at <= s["sees"][:, :, None])[None, :, :, None], -math.inf)
    top = near.amax(-1, keepdim=True)
    if prefix:
        top = torch.maximum(top, far.amax(-1, keepdim=True))
    top = torch.where(top.isinf(), torch.zeros_like(top), top)
    far, near = torch.exp(far - top), torch.exp(near - top)
    total = far.sum(-1, keepdim=True) + near.sum(-1, keepdim=True)
    out = (near.view(kv, n, most * group, width) @ tail[1].permute(2, 0, 1, 3)).view(kv, n, most, group, dim)
    out = out + (far.reshape(kv, n * most * group, prefix) @ shared[1].permute(1, 0, 2)).view(kv, n, most, group, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).permute(1, 2, 0, 3, 4).reshape(n, most, case["heads"], dim)
    s["out"][s["row"][s["live"]]] = out[s["live"]].to(s["out"].dtype)
    return s["out"]


def _run_verify(s):
    case = s["case"]
    if own:
        import rustyneedle_b200 as nb

        return nb.verify_drafts(s["logits"], s["tokens"], s["accept"], s["sample"], draft_probabilities=s["draft"], draft_counts=s["counts"],
                                mask_bits=s["mask"], temperature=case["temperature"])
    n, k, v = case["sequences"], case["drafts"], case["vocab"]
    x = s["logits"].double()  # probabilities and their running sums in 64 bits: a random number may lie next to a border
    if s["mask"] is not None:
        allowed = ((s["mask"][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).bool().view(n, k + 1, -1)[..., :v]
        x = torch.where(allowed | ~allowed.any(-1, keepdim=True), x, torch.full_like(x, -math.inf))
    drafted = s["tokens"].long()
    within = torch.arange(k, device="cuda")[None] < s["counts"][:, None]
    if case["temperature"] == 0:
        best = x.argmax(-1)
        good = (drafted == best[:, :k]) & within
        kept = good.long().cumprod(1).sum(1)
        last = best.gather(1, kept[:, None])[:, 0]
    else:
        p = torch.exp((x - x.amax(-1, keepdim=True)) / case["temperature"])
        p = p / p.sum(-1, keepdim=True)
        have = p[:, :k].gather(2, drafted[..., None])[..., 0]
        asked = s["draft"].gather(2, drafted[..., None])[..., 0].double() if case["given"] else torch.ones_like(have)
        good = (s["accept"].double() * asked < have) & within
        kept = good.long().cumprod(1).sum(1)
        rest = p.gather(1, kept[:, None, None].expand(n, 1, v))[:, 0]
        place = kept.clamp(max=k - 1)[:, None]
        if case["given"]:
            minus = s["draft"].gather(1, place[..., None].expand(n, 1, v))[:, 0].double()
        else:
            minus = torch.zeros_like(rest).scatter_(1, drafted.gather(1, place), 1.0)
        rejected = (kept < s["counts"])[:, None]
        left = torch.where(rejected, (rest - minus).clamp(min=0), rest)
        left = torch.where(left.sum(-1, keepdim=True) > 0, left, rest)
        upto = left.cumsum(-1)
        last = (upto > s["sample"].double()[:, None] * upto[:, -1:]).long().argmax(-1)
    place = torch.arange(k + 1, device="cuda")[None]
    padded = torch.cat([drafted, drafted[:, :1]], 1)
    tokens = torch.where(place < kept[:, None], padded, torch.where(place == kept[:, None], last[:, None], torch.full_like(padded, NONE)))
    return tokens.to(torch.int32), kept.to(torch.int32)


# ------------------------------------------------------------------------------------- the same from the definitions


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"cache": _exact_cache, "attend": _exact_attend, "verify": _exact_verify}[case["op"]](case, seed, s)


def _held(x, kind):
    """What a cache row holds of x, in 64 bits."""
    x = x.double()
    peak = x.abs().max(-1, keepdim=True).values
    peak = torch.where(peak == 0, torch.ones_like(peak), peak)
    if kind == "int8":
        step = (peak / 127).float().double()  # the scale itself is a 32-bit number
        return torch.round(x / step) * step
    scale = torch.exp2(torch.ceil(torch.log2(peak / 448)))
    y = x / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(y / step) * step * scale


def _exact_cache(case, seed, s):
    return _held(s["keys"], case["format"]), _held(s["values"], case["format"])


def _exact_attend(case, seed, s):
    rows, lengths, prefix = _rows(case), _lengths(case), case["prefix"]
    heads, kv, dim, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    if work(case)["flops"] > 2e11:
        return None
    g = _generator(seed)
    query, _, _ = _fused_rows(g, sum(rows), heads, kv, dim, dtype)
    query *= 0.6
    _, keys, values = _fused_rows(g, prefix + sum(lengths), 0, kv, dim, dtype)
    keys, values = _held(keys, case["format"]), _held(values, case["format"])
    out = torch.zeros(sum(rows), heads, dim, dtype=torch.float64, device="cuda")
    row, at = 0, prefix
    for r, t in zip(rows, lengths):
        for h in range(heads):
            j = h // (heads // kv)
            k = torch.cat([keys[:prefix, j], keys[at : at + t, j]])
            v = torch.cat([values[:prefix, j], values[at : at + t, j]])
            a = query[row : row + r, h].double() @ k.T / dim**0.5
            seen = torch.arange(prefix + t, device="cuda")[None] <= (prefix + t - r + torch.arange(r, device="cuda"))[:, None]
            out[row : row + r, h] = torch.softmax(torch.where(seen, a, torch.full_like(a, -math.inf)), -1) @ v
        row, at = row + r, at + t
    return out


def _exact_verify(case, seed, s):
    n, k, v, t = case["sequences"], case["drafts"], case["vocab"], case["temperature"]
    tokens = torch.full((n, k + 1), NONE, dtype=torch.int32)
    kept = torch.zeros(n, dtype=torch.int32)
    drafted, counts = s["tokens"].cpu(), s["counts"].cpu()
    accept, sample = s["accept"].double().cpu(), s["sample"].double().cpu()
    shift = torch.arange(32, device="cuda")
    for b in range(n):
        for i in range(int(counts[b]) + 1):
            x = s["logits"][b, i].double()
            if s["mask"] is not None:
                bits = ((s["mask"][b, i].long()[:, None] >> shift) & 1).view(-1)[:v].bool()
                if bool(bits.any()):
                    x[~bits] = -math.inf
            last = i == int(counts[b])
            d = 0 if last else int(drafted[b, i])
            if t == 0:
                best = int(torch.nonzero(x == x.max())[0])
                if not last and best == d:
                    tokens[b, i] = d
                    kept[b] += 1
                    continue
                tokens[b, i] = best
                break
            p = torch.softmax(x / t, 0)
            q = None
            if not last:
                q = s["draft"][b, i].double() if case["given"] else torch.nn.functional.one_hot(drafted[b, i].long(), v).double().cuda()
                if float(accept[b, i]) * float(q[d]) < float(p[d]):
                    tokens[b, i] = d
                    kept[b] += 1
                    continue
            left = p if q is None else torch.relu(p - q)
            left = left if float(left.sum()) > 0 else p
            upto = torch.cumsum(left, 0)
            tokens[b, i] = int(torch.searchsorted(upto, upto[-1] * float(sample[b]), right=True).clamp(max=v - 1))
            break
    return tokens.cuda(), kept.cuda()
