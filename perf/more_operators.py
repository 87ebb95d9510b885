"""Performance cases of attention over selected blocks of a key-value cache: the blocks' summaries, the
selection that a cheap score makes for each query, the attention over what was selected, and its gradients.

A case names an entry point (`call`), its sizes and its types.  `prepare` makes the operands on the GPU from
the seed and the sequences' description that a program keeps; `run` is one pass; `exact` is the same from the
definition in 64 bits.

Entry points (`call`):
  means           flagsparse_block_means: the mean of each block's keys
  select          flagsparse_block_select: per query and key-value head the blocks with the largest scores
  attention       flagsparse_block_attention: softmax over the keys of those blocks, times their values
  attention_grad  flagsparse_block_attention_grad: its gradients in queries, keys and values

Sequences: `sequences` of them, of `context` keys and fewer (the first of all, the others down to half);
`new` of each one's last positions are queries, 0 for all (a prompt, a training batch).  `page` > 0 takes the
keys from a cache in pages of that many rows, in any order; 0 from packed rows.  A group of `group` query
heads shares a key-value head and its selection.  Queries and keys drift: positions near each other have a
part in common, so that neighbouring queries select many of the same blocks, and far ones others.
"""

import math

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # one decode step: the block that each sequence's new key fell into
        dict(name="means_append_64_bf16", call="means", sequences=64, new=1, context=16384, page=64, kv_heads=8,
             width=128, block=64, dtype="bf16"),
        # a batch of prompts' summaries
        dict(name="means_prompts_8x16k_f16", call="means", sequences=8, new=0, context=16384, page=0, kv_heads=8,
             width=128, block=64, dtype="f16"),
        # a decode step of a batch over long contexts: the summaries' bytes are what counts
        dict(name="select_decode_32_bf16", call="select", sequences=32, new=1, context=65536, page=64, kv_heads=8,
             group=4, width=128, block=64, top=16, dtype="bf16"),
        # a long prompt
        dict(name="select_16k_bf16", call="select", sequences=1, new=0, context=16384, page=0, kv_heads=4, group=16,
             width=128, block=64, top=16, dtype="bf16"),
        # a chunk of new tokens, odd sizes, 32-bit values
        dict(name="select_odd_f32", call="select", sequences=3, new=333, context=20011, page=0, kv_heads=2, group=5,
             width=80, block=32, top=24, dtype="f32"),
        # one sequence's next token: latency
        dict(name="attention_1_bf16", call="attention", sequences=1, new=1, context=8192, page=64, kv_heads=8,
             group=4, width=128, block=64, top=16, dtype="bf16"),
        # a decode step of a batch
        dict(name="attention_decode_64_bf16", call="attention", sequences=64, new=1, context=16384, page=64,
             kv_heads=8, group=8, width=128, block=64, top=16, dtype="bf16"),
        # chunks of new tokens of several sequences over a cache of small pages
        dict(name="attention_chunk_4x512_f16", call="attention", sequences=4, new=512, context=16384, page=16,
             kv_heads=4, group=8, width=128, block=64, top=32, dtype="f16"),
        # a long prompt: the largest case
        dict(name="attention_16k_bf16", call="attention", sequences=1, new=0, context=16384, page=0, kv_heads=4,
             group=16, width=128, block=64, top=16, dtype="bf16"),
        # odd lengths and widths, small blocks, 32-bit values
        dict(name="attention_odd_f32", call="attention", sequences=3, new=0, context=2501, page=0, kv_heads=4,
             group=3, width=80, block=32, top=8, dtype="f32"),
        # a training sequence
        dict(name="attention_grad_8k_bf16", call="attention_grad", sequences=1, new=0, context=8192, page=0,
             kv_heads=4, group=8, width=128, block=64, top=16, dtype="bf16"),
        # a training batch of unlike sequences without shared heads
        dict(name="attention_grad_odd_f16", call="attention_grad", sequences=5, new=0, context=1501, page=0,
             kv_heads=8, group=1, width=64, block=32, top=12, dtype="f16"),
    ]


_MAX_GATHERED = 1 << 33  # selected keys' values of all queries and key-value heads, the largest listed case's
_MAX_PAIRS = 1 << 31  # queries x keys x heads of a gradient, the largest listed case's
_MAX_KEYS = 1 << 29  # values of all keys


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    call = rng.choice(["means", "select", "attention", "attention", "attention_grad", "attention_grad"])
    case = dict(call=call, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), kv_heads=rng.choice([1, 2, 4, 8]),
                block=rng.choice([32, 64, 64, 128]))
    case["width"] = rng.choice([32, 64, 80, 96, 128, 128, 128] + ([] if case["dtype"] == "f32" else [256]))
    per_key = case["kv_heads"] * case["width"]
    if call != "means":
        case["group"] = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        case["top"] = rng.choice([4, 8, 16, 24, 32] + ([] if call == "select" else [2]))
    # a selection is one where a context has more blocks than it takes
    least = (case["top"] + 8) * case["block"] if call == "select" else 8
    if call == "attention_grad":
        case["new"] = case["page"] = 0
        most = math.isqrt(_MAX_PAIRS // (case["kv_heads"] * case["group"]))
        case["sequences"] = _log_int(rng, 1, 16)
        case["context"] = _log_int(rng, 16, max(16, min(8192, most // case["sequences"])))
        return case
    case["page"] = rng.choice([0, 16, 64, 256])
    case["new"] = rng.choice([0, 1, 1, 4]) if rng.random() < 0.7 else _log_int(rng, 2, 1024)
    if case["new"] == 0:
        case["sequences"] = _log_int(rng, 1, 16)
        most = min(65536, _MAX_KEYS // (per_key * case["sequences"]))
        if call == "attention":
            most = min(most, _MAX_GATHERED // (case["sequences"] * per_key * case["top"] * case["block"]))
        if call == "select":
            most = min(most, math.isqrt((1 << 28) // (case["sequences"] * case["kv_heads"]) * case["block"]))
        case["context"] = _log_int(rng, least, max(least, most))
        return case
    case["context"] = _log_int(rng, max(least, case["new"]), 131072)
    most = min(256, _MAX_KEYS // (per_key * case["context"]))
    if call == "attention":
        most = min(most, _MAX_GATHERED // (case["new"] * per_key * case["top"] * case["block"]))
    if call == "select":
        most = min(most, (1 << 28) // (case["new"] * case["kv_heads"] * (case["context"] // case["block"] + 1)))
    case["sequences"] = _log_int(rng, 1, max(1, most))
    return case


def _lengths(case):
    """Each sequence's keys, and how many of them are new: the first has all of `context`."""
    lengths = []
    for i in range(case["sequences"]):
        part = 1.0 - 0.5 * ((i * 0.6180339887) % 1.0)
        lengths.append(max(1, case["new"], int(case["context"] * part)))
    return lengths, [case["new"] or n for n in lengths]


def work(case):
    """Inputs once, outputs once; of a cache, what is selected (at most all of it)."""
    lengths, new = _lengths(case)
    s, heads, width, block = _BYTES[case["dtype"]], case["kv_heads"], case["width"], case["block"]
    row = heads * width * s
    if case["call"] == "means":
        keys = blocks = 0
        for n, m in zip(lengths, new):
            first = (n - m) // block
            keys += n - first * block
            blocks += -(-n // block) - first
        return {"bytes": (keys + blocks) * row, "flops": keys * heads * width}
    group, top = case["group"], case["top"]
    tokens, seen, reads, scored, summaries, chosen = sum(new), 0, 0, 0, 0, 0
    for n, m in zip(lengths, new):
        here = 0
        for p in range(n - m, n):
            blocks = min(top, p // block + 1)
            here += (blocks - 1) * block + p % block + 1
            chosen += blocks
            scored += p // block + 1
        seen += here
        reads += min(here, n)
        summaries += -(-n // block)
    q = tokens * heads * group * width * s
    if case["call"] == "select":
        return {"bytes": q + summaries * row + 4 * tokens * heads * top,
                "flops": 2 * scored * heads * width + tokens * heads * group * width}
    keys = 2 * reads * row + 4 * chosen * heads
    if case["call"] == "attention":
        return {"bytes": 2 * q + keys, "flops": 4 * seen * heads * group * width}
    return {"bytes": 4 * q + 2 * 2 * sum(lengths) * row + 4 * tokens * heads * (top + group),
            "flops": 10 * seen * heads * group * width}


# -- inputs ----------------------------------------------------------------------------


def _drifting(rows, heads, width, span, gen):
    """Normal values, half as large a part of which rows of the same `span` have in common."""
    common = torch.randn((rows // span + 2, heads, width), device="cuda", generator=gen)
    out = torch.randn((rows, heads, width), device="cuda", generator=gen)
    at = torch.arange(rows, device="cuda") // span
    return out.add_(common[at], alpha=0.5)


def _positions(lengths, new):
    """Of each query: its sequence and its position, on the GPU."""
    lengths, new = (torch.tensor(x, device="cuda") for x in (lengths, new))
    seq = torch.repeat_interleave(torch.arange(new.numel(), device="cuda"), new)
    first = torch.cumsum(new, 0) - new
    return seq, torch.arange(seq.numel(), device="cuda") - first[seq] + (lengths - new)[seq]


def _offsets(counts):
    out = torch.zeros(len(counts) + 1, dtype=torch.int32)
    out[1:] = torch.cumsum(torch.tensor(counts), 0)
    return out.cuda()


def _operands(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    call, dtype = case["call"], _DTYPES[case["dtype"]]
    lengths, new = _lengths(case)
    heads, width, block, page = case["kv_heads"], case["width"], case["block"], case["page"]
    a = dict(q_offsets=_offsets(new), k_lengths=torch.tensor(lengths, dtype=torch.int32).cuda())
    total, most = sum(lengths), -(-max(lengths) // block)
    if call == "select":
        means = _drifting(len(lengths) * most, heads, width, 2, gen) * 0.5
        a["means"] = means.view(len(lengths), most, heads, width).to(dtype)
    else:
        k = _drifting(total, heads, width, 128, gen).to(dtype)
        if page:
            per = [-(-n // page) for n in lengths]
            ids = torch.randperm(sum(per) + 3, device="cuda", generator=gen)[: sum(per)].int()
            pages = torch.full((len(lengths), max(per)), -1, dtype=torch.int32, device="cuda")
            at = 0
            for i, n in enumerate(per):
                pages[i, :n] = ids[at : at + n]
                at += n
            a["pages"] = pages
            seq, pos = _positions(lengths, lengths)
            slots = pages[seq, pos // page].long() * page + pos % page
        def laid(rows):
            if not page:
                return rows
            cache = torch.zeros(((sum(per) + 3) * page, heads, width), dtype=dtype, device="cuda")
            cache[slots] = rows
            return cache.view(-1, page, heads, width)
        if call != "means":
            a["v"] = laid(torch.randn((total, heads, width), device="cuda", generator=gen).to(dtype))
            summaries = torch.zeros((len(lengths) * most, heads, width), device="cuda")
            seq, pos = _positions(lengths, lengths)
            summaries.index_add_(0, seq * most + pos // block, k.float())
            a["summaries"] = (summaries / block).view(len(lengths), most, heads, width)
        a["k"] = laid(k)
    if not page:
        a["k_offsets"] = _offsets(lengths)
    if call == "means":
        a["most"] = most
        return a
    group, tokens = case["group"], sum(new)
    q = _drifting(tokens, heads * group, width, 256, gen)
    a["q"] = q.to(dtype)
    if call.startswith("attention"):
        # the selection that a program would have made before
        seq, pos = _positions(lengths, new)
        a["blocks"] = _plain_select(a["q"], a.pop("summaries"), seq, pos, case)
    if call == "attention_grad":
        a["grad"] = torch.randn(q.shape, device="cuda", generator=gen).to(dtype)
    return a


def prepare(case, seed):
    a = _operands(case, seed)
    lengths, new = _lengths(case)
    state = dict(a, call=case["call"], case=case, scale=case["width"] ** -0.5)
    if own:
        import flagsparse_amd as fs

        # (the selection reads no keys, only how many there are)
        paged = "pages" in a
        state["seqs"] = fs.prepare_block_sequences(case["block"], q_offsets=a["q_offsets"],
                                                   k_offsets=None if paged else _offsets(lengths),
                                                   pages=a.get("pages"), k_lengths=a["k_lengths"] if paged else None)
    else:
        state["seq"], state["pos"] = _positions(lengths, new)
    if case["call"] == "means":
        state["start"] = a["k_lengths"] - torch.tensor(new, dtype=torch.int32).cuda()
        state["means"] = torch.zeros((len(lengths), a["most"], case["kv_heads"], case["width"]),
                                     dtype=a["k"].dtype, device="cuda")
        state["touched"] = max(-(-n // case["block"]) - (n - m) // case["block"] for n, m in zip(lengths, new))
    if case["call"] == "attention_grad":
        # the forward pass's results, kept for the backward pass
        state["seq"], state["pos"] = _positions(lengths, new)
        state["out"], state["lse"] = _plain_attention(state)
    return state


# -- one pass --------------------------------------------------------------------------


def _run_own(s):
    import flagsparse_amd as fs

    call, seqs = s["call"], s["seqs"]
    if call == "means":
        return fs.flagsparse_block_means(s["k"], seqs, start=s["start"], out=s["means"])
    if call == "select":
        return fs.flagsparse_block_select(s["q"], s["means"], seqs, s["case"]["top"])
    if call == "attention":
        return fs.flagsparse_block_attention(s["q"], s["k"], s["v"], s["blocks"], seqs, scale=s["scale"])
    return fs.flagsparse_block_attention_grad(s["grad"], s["q"], s["k"], s["v"], s["blocks"], seqs, s["out"], s["lse"],
                                              scale=s["scale"])


def _rows(s, seq, pos):
    """Rows of the keys at positions of sequences, in the packed rows or the cache's."""
    page = s["case"]["page"]
    if page:
        return s["pages"][seq, pos // page].long() * page + pos % page
    return s["k_offsets"][seq].long() + pos


def _plain_select(q, means, seq, pos, case):
    """The first block, the query's own, and of the others before it those of the largest scores; ties to the
    lowest, the result ascending, -1 behind it.  Scores in 64 bits: two of them near each other decide."""
    block, top, most = case["block"], case["top"], means.shape[1]
    tokens, heads = q.shape[0], means.shape[2]
    # each sequence's queries side by side
    index = pos - torch.full_like(pos, 1 << 40).scatter_reduce_(0, seq, pos, "amin")[seq]
    side = torch.zeros((means.shape[0], case["new"] or case["context"], heads, q.shape[2]), dtype=torch.float64,
                       device="cuda")
    side[seq, index] = q.view(tokens, heads, -1, q.shape[2]).double().sum(2)
    score = torch.matmul(side.transpose(1, 2).contiguous(), means.double().permute(0, 2, 3, 1).contiguous())
    score = score[seq, :, index]
    ids = torch.arange(most, device="cuda")
    mine = (pos // block)[:, None, None]
    score = torch.where(ids < mine, score, -math.inf)
    score = torch.where(((ids == 0) & (ids <= mine)) | (ids == mine), math.inf, score)
    best, at = torch.sort(score, dim=2, descending=True, stable=True)
    at = torch.where(best[:, :, :top] > -math.inf, at[:, :, :top], most)
    at = torch.sort(at, dim=2)[0]
    at = torch.nn.functional.pad(at, (0, top - at.shape[2]), value=most)
    return torch.where(at < most, at, -1).int()


def _plain_attention(s):
    """Every query's selected keys gathered."""
    case, q, blocks = s["case"], s["q"], s["blocks"].long()
    tokens, heads, top = blocks.shape
    block, group, width = case["block"], case["group"], case["width"]
    at = (blocks[:, :, :, None] * block + torch.arange(block, device="cuda")).view(tokens, heads, top * block)
    seen = (blocks >= 0).repeat_interleave(block, dim=2) & (at <= s["pos"][:, None, None])
    rows = _rows(s, s["seq"][:, None, None], torch.where(seen, at, 0))
    head = torch.arange(heads, device="cuda")[None, :, None]
    keys = s["k"].view(-1, heads, width)[rows, head].float()
    score = torch.matmul(q.view(tokens, heads, group, width).float(), keys.transpose(2, 3)) * s["scale"]
    del keys
    score = torch.where(seen[:, :, None], score, -math.inf)
    top_score = score.amax(3, keepdim=True)
    weight = torch.exp(score - top_score)
    total = weight.sum(3, keepdim=True)
    values = s["v"].view(-1, heads, width)[rows, head].float()
    out = torch.matmul(weight, values) / total
    lse = (top_score + torch.log(total)).view(tokens, heads * group)
    return out.reshape(q.shape).to(q.dtype), lse


def _plain_grad(s):
    """All pairs of queries and keys, masked."""
    case, seq, pos = s["case"], s["seq"], s["pos"]
    heads, group, width, block = case["kv_heads"], case["group"], case["width"], case["block"]
    tokens, most = s["q"].shape[0], int(case["context"]) // block + 2
    chosen = torch.zeros((tokens, heads, most + 1), dtype=torch.bool, device="cuda")
    chosen.scatter_(2, torch.where(s["blocks"] >= 0, s["blocks"], most).long(), True)
    seen = chosen.transpose(0, 1)[:, :, pos // block] & (seq[:, None] == seq) & (pos[:, None] >= pos)
    def by_head(x):
        return x.view(tokens, heads, group, width).permute(1, 2, 0, 3).float().reshape(heads, group * tokens, width)
    q, grad, out = by_head(s["q"]), by_head(s["grad"]), by_head(s["out"])
    k, v = (s[n].transpose(0, 1).float().contiguous() for n in ("k", "v"))
    score = torch.matmul(q, k.transpose(1, 2)) * s["scale"]
    lse = s["lse"].view(tokens, heads, group).permute(1, 2, 0).reshape(heads, group * tokens, 1)
    weight = torch.exp(score - lse)
    del score
    weight = torch.where(seen[:, None], weight.view(heads, group, tokens, tokens), 0.0).view(heads, -1, tokens)
    grad_v = torch.matmul(weight.transpose(1, 2), grad)
    inner = torch.matmul(grad, v.transpose(1, 2)) - (grad * out).sum(2, keepdim=True)
    inner = weight * inner * s["scale"]
    grad_q = torch.matmul(inner, k).view(heads, group, tokens, width).permute(2, 0, 1, 3)
    grad_k = torch.matmul(inner.transpose(1, 2), q)
    dtype = s["q"].dtype
    return (grad_q.reshape(s["q"].shape).to(dtype), grad_k.transpose(0, 1).contiguous().to(dtype),
            grad_v.transpose(0, 1).contiguous().to(dtype))


def _plain_means(s):
    """The blocks that hold a key from `start` on, in the summaries that the program keeps."""
    case, means = s["case"], s["means"]
    block, n = case["block"], means.shape[0]
    lengths = s["k_lengths"].long()
    ids = (s["start"].long() // block)[:, None] + torch.arange(s["touched"], device="cuda")
    at = ids[:, :, None] * block + torch.arange(block, device="cuda")
    here = at < lengths[:, None, None]
    seq = torch.arange(n, device="cuda")
    rows = _rows(s, seq[:, None, None], torch.where(here, at, 0))
    keys = torch.where(here[:, :, :, None, None], s["k"].view(-1, *means.shape[2:])[rows].float(), 0.0)
    mean = keys.sum(2) / here.sum(2)[:, :, None, None].clamp(min=1)
    inside = ids * block < lengths[:, None]
    seq = seq[:, None].expand_as(ids)[inside]
    means[seq, ids[inside]] = mean[inside].to(means.dtype)
    return means


def run(s):
    if own:
        return _run_own(s)
    if s["call"] == "means":
        return _plain_means(s)
    if s["call"] == "select":
        return _plain_select(s["q"], s["means"], s["seq"], s["pos"], s["case"])
    if s["call"] == "attention":
        return _plain_attention(s)[0]
    return _plain_grad(s)


# -- reference -------------------------------------------------------------------------


def _sequence(case, a, name, i, lengths):
    """Rows of one sequence's keys or values, in order."""
    n, x = lengths[i], a[name]
    if case["page"]:
        page = case["page"]
        return x[a["pages"][i, : -(-n // page)].long()].reshape(-1, *x.shape[2:])[:n].double()
    first = sum(lengths[:i])
    return x[first : first + n].double()


def exact(case, seed):
    """The definitions in 64 bits, one sequence and head after the other, over all its keys with what is not
    selected left out; the gradients by differentiating that."""
    a = _operands(case, seed)
    lengths, new = _lengths(case)
    call, heads, width, block = case["call"], case["kv_heads"], case["width"], case["block"]
    if call == "means":
        out = torch.zeros((len(lengths), a["most"], heads, width), dtype=torch.float64, device="cuda")
        for i, n in enumerate(lengths):
            keys = _sequence(case, a, "k", i, lengths)
            first = (n - new[i]) // block
            full = n // block
            if full > first:
                out[i, first:full] = keys[first * block : full * block].view(-1, block, heads, width).mean(1)
            if n % block:
                out[i, full] = keys[full * block :].mean(0)
        return out
    group, top, tokens = case["group"], case["top"], sum(new)
    if call == "select":
        out = torch.full((tokens, heads, top), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(lengths):
            for h in range(heads):
                q = a["q"][at : at + new[i], h * group : (h + 1) * group].double().sum(1)
                mine = torch.arange(n - new[i], n, device="cuda") // block
                score = q @ a["means"][i, :, h].double().T
                ids = torch.arange(score.shape[1], device="cuda")
                score[ids[None] > mine[:, None]] = -math.inf
                score[:, 0] = math.inf
                score[ids[None] == mine[:, None]] = math.inf
                order = torch.sort(-score, dim=1, stable=True)[1]
                rank = torch.empty_like(order)
                rank.scatter_(1, order, ids.expand_as(order))
                taken = (rank < top) & (ids[None] <= mine[:, None])
                place = torch.cumsum(taken, 1) - 1
                t, b = torch.nonzero(taken, as_tuple=True)
                out[at + t, h, place[t, b]] = b.int()
            at += new[i]
        return out
    outs = torch.zeros((tokens, heads * group, width), dtype=torch.float64, device="cuda")
    grads = [torch.zeros(a[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v")] \
        if call == "attention_grad" else None
    at = 0
    for i, n in enumerate(lengths):
        keys, values = (_sequence(case, a, x, i, lengths) for x in ("k", "v"))
        mine = torch.arange(n - new[i], n, device="cuda")
        for h in range(heads):
            here = slice(at, at + new[i])
            named = torch.zeros((new[i], -(-n // block) + 1), dtype=torch.bool, device="cuda")
            ids = a["blocks"][here, h].long()
            named.scatter_(1, torch.where(ids < 0, named.shape[1] - 1, ids), True)
            step = max(1, (1 << 28) // (n * group))
            cols = slice(h * group, (h + 1) * group)
            for t in range(0, new[i], step):
                part = slice(t, min(t + step, new[i]))
                rows = slice(at + part.start, at + part.stop)
                hidden = ~named[part][:, torch.arange(n, device="cuda") // block]
                hidden |= torch.arange(n, device="cuda")[None] > mine[part, None]
                leaves = [x.detach().requires_grad_(grads is not None)
                          for x in (a["q"][rows, cols].double(), keys[:, h], values[:, h])]
                with torch.set_grad_enabled(grads is not None):
                    score = torch.matmul(leaves[0].transpose(0, 1), leaves[1].T) / math.sqrt(width)
                    weight = torch.softmax(score.masked_fill(hidden, -math.inf), 2)
                    out = torch.matmul(weight, leaves[2]).transpose(0, 1)
                if grads is None:
                    outs[rows, cols] = out
                    continue
                d = torch.autograd.grad(out, leaves, a["grad"][rows, cols].double())
                grads[0][rows, cols] = d[0]
                first = sum(lengths[:i])
                grads[1][first : first + n, h] += d[1]
                grads[2][first : first + n, h] += d[2]
        at += new[i]
    return outs if grads is None else tuple(grads)
