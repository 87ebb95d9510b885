"""Performance cases of the products with selection matrices: embedding lookup and the routing
of tokens to experts, with the experts' products between sorting and sorting back.

A case names an entry point (`call`), its sizes and its types.  `prepare` makes the operands on
the GPU from the seed, plus the route where a program keeps one; `run` is one pass; `exact` is
the same from the definition in 64 bits.

Entry points (`call`):
  embedding        flagsparse_embedding: table rows of the tokens, scaled
  embedding_grad   flagsparse_embedding_grad: the table's gradient
  route            prepare_expert_route: tokens' slots sorted by expert
  dispatch         flagsparse_expert_dispatch: token rows into expert order
  dispatch_grad    flagsparse_expert_dispatch_grad: its gradient
  combine          flagsparse_expert_combine: expert rows back, weighted and summed
  combine_grad     flagsparse_expert_combine_grad: gradients of the rows and of the weights
  product          flagsparse_expert_product: each row times its expert's matrix
  product_grad     flagsparse_expert_product_grad: gradients of the rows and of the matrices

Tokens follow a Zipf law (exponent 1) over a shuffled vocabulary; experts' popularities are
log-normal, each token takes distinct experts, and a share `dropped` of the slots names none
(over capacity, or an expert of another process).
"""

import math

import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_INDEX = {"i32": torch.int32, "i64": torch.int64}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4, "i32": 4, "i64": 8}


def listed():
    return [
        # one sequence's next token: the launch and the call are what counts
        dict(name="embedding_1_bf16", call="embedding", tokens=1, vocab=32768, width=4096, dtype="bf16", index="i64",
             scale=64.0),
        # a training batch's or a long prompt's lookup in a large vocabulary
        dict(name="embedding_32k_bf16", call="embedding", tokens=32768, vocab=131072, width=4096, dtype="bf16",
             index="i64", scale=64.0),
        # a small model's gradient, odd sizes, 32-bit values
        dict(name="embedding_grad_4095_f32", call="embedding_grad", tokens=4095, vocab=20011, width=1001, dtype="f32",
             index="i32", scale=1.0),
        # a large batch's gradient: frequent tokens occur thousands of times, most of the vocabulary never
        dict(name="embedding_grad_64k_bf16", call="embedding_grad", tokens=65536, vocab=131072, width=2048,
             dtype="bf16", index="i64", scale=45.25),
        # a decode step of a batch of sequences: slots sorted by expert
        dict(name="route_64x8", call="route", tokens=64, slots=8, experts=64, index="i32", dropped=0.0),
        # a training batch, some slots over capacity
        dict(name="route_128k_x8", call="route", tokens=131072, slots=8, experts=128, index="i64", dropped=0.03),
        # a decode step's way back
        dict(name="combine_16x4_bf16", call="combine", tokens=16, slots=4, experts=32, width=2048, dtype="bf16",
             dropped=0.0),
        # a prompt's or training batch's rows into expert order
        dict(name="dispatch_16k_x8_bf16", call="dispatch", tokens=16384, slots=8, experts=64, width=2048, dtype="bf16",
             dropped=0.02),
        # the backward step of the way back, an odd number of tokens
        dict(name="combine_grad_8191x8_f16", call="combine_grad", tokens=8191, slots=8, experts=64, width=2560,
             dtype="f16", dropped=0.02),
        # a decode step's experts: a few rows each, the matrices' bytes are what counts
        dict(name="product_16x4_bf16", call="product", tokens=16, slots=4, experts=32, inner=2048, outer=4096,
             dtype="bf16", op="trans", dropped=0.0),
        # a training batch's experts: the largest case
        dict(name="product_16k_x2_bf16", call="product", tokens=16384, slots=2, experts=16, inner=4096, outer=4096,
             dtype="bf16", op="non", dropped=0.0),
        # both gradients of a batch with an odd number of tokens
        dict(name="product_grad_4093x4_f16", call="product_grad", tokens=4093, slots=4, experts=8, inner=2048,
             outer=5120, dtype="f16", op="trans", dropped=0.02),
    ]


_MAX_FLOPS = 1 << 39  # an expert product's, half of the largest listed case's
_MAX_VALUES = 1 << 28  # of the largest operand of the other calls


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly whole 16-byte pieces, as models have them; one in five at random."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.2 else max(8, n // 8 * 8)


def draw(rng):
    call = rng.choice(["embedding", "embedding_grad", "route", "dispatch", "dispatch_grad", "combine", "combine_grad",
                       "product", "product", "product_grad"])
    case = dict(call=call)
    if call != "route":
        case["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
    if call.startswith("embedding"):
        width = case["width"] = _width(rng, 64, 8192)
        case["index"] = rng.choice(["i32", "i64"])
        case["vocab"] = _log_int(rng, 1000, min(262144, _MAX_VALUES // width))
        case["tokens"] = _log_int(rng, 1, min(131072, _MAX_VALUES // width))
        case["scale"] = rng.choice([1.0, 0.5, round(math.sqrt(width), 2)])
        return case
    case["experts"] = rng.choice([4, 8, 16, 32, 60, 64, 128, 256])
    slots = case["slots"] = rng.choice([n for n in (1, 2, 4, 6, 8) if n <= case["experts"]])
    case["dropped"] = rng.choice([0.0, 0.0, 0.02, 0.1])
    if call == "route":
        case["index"] = rng.choice(["i32", "i64"])
        case["tokens"] = _log_int(rng, 1, 262144)
        return case
    if not call.startswith("product"):
        width = case["width"] = _width(rng, 128, 8192)
        case["tokens"] = _log_int(rng, 1, min(65536, _MAX_VALUES // (width * slots)))
        return case
    case["op"] = rng.choice(["non", "trans"])
    case["inner"], case["outer"] = _width(rng, 256, 6000), _width(rng, 256, 6000)
    area = case["inner"] * case["outer"]
    while case["experts"] > 8 and case["experts"] * area > 1 << 30:
        case["experts"] //= 2
    case["slots"] = slots = min(slots, case["experts"])
    passes = (4 if call == "product_grad" else 2) * (8 if case["dtype"] == "f32" else 1)
    case["tokens"] = _log_int(rng, 1, max(2, min(32768, _MAX_FLOPS // (passes * area * slots))))
    return case


def _zipf(vocab):
    p = 1.0 / torch.arange(1, vocab + 1, dtype=torch.float64)
    return p / p.sum()


def work(case):
    """Inputs once, outputs once: of tables and matrices what the tokens are expected to touch."""
    call, n = case["call"], case["tokens"]
    if call.startswith("embedding"):
        s, width = _BYTES[case["dtype"]], case["width"]
        ids = n * _BYTES[case["index"]]
        if call == "embedding":
            touched = float((1.0 - (1.0 - _zipf(case["vocab"])) ** n).sum())
            return {"bytes": int(ids + (touched + n) * width * s), "flops": n * width}
        return {"bytes": ids + (n + case["vocab"]) * width * s, "flops": n * width}
    rows = n * case["slots"]
    if call == "route":
        return {"bytes": rows * (_BYTES[case["index"]] + 8) + 4 * (case["experts"] + 1), "flops": rows}
    s = _BYTES[case["dtype"]]
    places = 4 * rows
    if call.startswith("product"):
        k, f, e = case["inner"], case["outer"], case["experts"]
        if call == "product":
            chosen = e * (1.0 - (1.0 - case["slots"] / e) ** n)
            return {"bytes": int((rows * (k + f) + chosen * k * f) * s), "flops": 2 * rows * k * f}
        return {"bytes": (rows * (2 * k + f) + 2 * e * k * f) * s, "flops": 4 * rows * k * f}
    width = case["width"]
    if call == "combine_grad":
        return {"bytes": (2 * rows + n) * width * s + 2 * 4 * rows + places, "flops": 3 * rows * width}
    return {"bytes": (rows + n) * width * s + places + (4 * rows if call == "combine" else 0), "flops": rows * width}


# -- inputs ----------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(shape, dtype, g, scale=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat, step = out.view(-1), 1 << 27
    for a in range(0, flat.numel(), step):
        part = flat[a : a + step]
        part.copy_(torch.randn(part.numel(), device="cuda", generator=g) * scale)
    return out


def _tokens(case, g):
    """Zipf: the inverse of the law's distribution function at uniform points."""
    vocab = case["vocab"]
    edges = torch.cumsum(_zipf(vocab).cuda(), 0)
    u = torch.rand(case["tokens"], dtype=torch.float64, device="cuda", generator=g)
    rank = torch.searchsorted(edges, u).clamp_(max=vocab - 1)
    return torch.randperm(vocab, device="cuda", generator=g)[rank].to(_INDEX[case["index"]])


def _experts(case, g):
    """Distinct experts a token (the largest of noise plus log popularity); -1 or E where a slot names none."""
    e, shape = case["experts"], (case["tokens"], case["slots"])
    popularity = torch.randn(e, device="cuda", generator=g) * 0.5
    u = torch.rand((case["tokens"], e), device="cuda", generator=g).clamp_(min=1e-9, max=1 - 1e-6)
    experts = torch.topk(popularity - torch.log(-torch.log(u)), case["slots"], dim=1)[1]
    if case["dropped"]:
        u = torch.rand(shape, device="cuda", generator=g)
        experts = torch.where(u < case["dropped"], torch.where(u < case["dropped"] / 2, -1, e), experts)
    return experts.to(_INDEX[case.get("index", "i32")])


def _operands(case, seed):
    """The call's own arguments, route aside."""
    g = _generator(seed)
    call = case["call"]
    if call.startswith("embedding"):
        rows = case["vocab"] if call == "embedding" else case["tokens"]
        return dict(tokens=_tokens(case, g), values=_randn((rows, case["width"]), _DTYPES[case["dtype"]], g))
    a = dict(experts=_experts(case, g))
    if call == "route":
        return a
    n, slots, dtype = case["tokens"], case["slots"], _DTYPES[case["dtype"]]
    if call.startswith("product"):
        k, f = case["inner"], case["outer"]
        shape = (case["experts"], k, f) if case["op"] == "non" else (case["experts"], f, k)
        a["rows"] = _randn((n * slots, k), dtype, g)
        a["matrices"] = _randn(shape, dtype, g, k**-0.5)
        if call == "product_grad":
            a["grad"] = _randn((n * slots, f), dtype, g)
        return a
    if call in ("dispatch", "combine_grad"):
        a["tokens"] = _randn((n, case["width"]), dtype, g)
    if call != "dispatch":
        a["rows"] = _randn((n * slots, case["width"]), dtype, g)
    if call.startswith("combine"):
        a["weights"] = torch.softmax(torch.randn((n, slots), device="cuda", generator=g), 1)
    return a


def _plain_route(experts, n_experts):
    flat = experts.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < n_experts), flat, n_experts)
    order = torch.sort(key, stable=True)[1]
    inverse = torch.empty_like(order)
    inverse[order] = torch.arange(order.numel(), device=order.device)
    counts = (key[:, None] == torch.arange(n_experts, device=key.device)).sum(0) if key.numel() * n_experts < 1 << 28 \
        else torch.bincount(key, minlength=n_experts + 1)[:n_experts]
    offsets = torch.zeros(n_experts + 1, dtype=torch.int64, device=key.device)
    offsets[1:] = torch.cumsum(counts, 0)
    return order, inverse.reshape(experts.shape), offsets


def prepare(case, seed):
    state = dict(case, **_operands(case, seed))
    if "experts" in case:
        state["n_experts"] = case["experts"]
        if case["call"] != "route":
            if own:
                import flagsparse_amd as fs

                state["route"] = fs.prepare_expert_route(state["experts"], case["experts"])
            else:
                order, inverse, offsets = _plain_route(state["experts"], case["experts"])
                state.update(order=order, inverse=inverse, bounds=offsets.tolist())
    if case["call"].startswith("embedding"):
        state["ids"], state["n_rows"] = state.pop("tokens"), case["vocab"]
    return state


# -- one pass --------------------------------------------------------------------------


def _run_own(s):
    import flagsparse_amd as fs

    call = s["call"]
    if call == "embedding":
        return fs.flagsparse_embedding(s["values"], s["ids"], scale=s["scale"])
    if call == "embedding_grad":
        return fs.flagsparse_embedding_grad(s["values"], s["ids"], s["n_rows"], scale=s["scale"])
    if call == "route":
        route = fs.prepare_expert_route(s["experts"], s["n_experts"])
        return route.order, route.inverse, route.offsets
    if call == "dispatch":
        return fs.flagsparse_expert_dispatch(s["tokens"], s["route"])
    if call == "dispatch_grad":
        return fs.flagsparse_expert_dispatch_grad(s["rows"], s["route"])
    if call == "combine":
        return fs.flagsparse_expert_combine(s["rows"], s["route"], s["weights"])
    if call == "combine_grad":
        return fs.flagsparse_expert_combine_grad(s["tokens"], s["rows"], s["route"], s["weights"])
    if call == "product":
        return fs.flagsparse_expert_product(s["rows"], s["matrices"], s["route"], op=s["op"])
    return fs.flagsparse_expert_product_grad(s["grad"], s["rows"], s["matrices"], s["route"], op=s["op"])


def run(s):
    if own:
        return _run_own(s)
    call = s["call"]
    if call == "embedding":
        inside = (s["ids"] >= 0) & (s["ids"] < s["values"].shape[0])
        rows = s["values"][torch.where(inside, s["ids"], 0).long()].float() * s["scale"]
        return torch.where(inside[:, None], rows, 0.0).to(s["values"].dtype)
    if call == "embedding_grad":
        inside = (s["ids"] >= 0) & (s["ids"] < s["n_rows"])
        rows = torch.where(inside[:, None], s["values"].float() * s["scale"], 0.0)
        out = torch.zeros((s["n_rows"], s["values"].shape[1]), device="cuda")
        return out.index_add_(0, torch.where(inside, s["ids"], 0).long(), rows).to(s["values"].dtype)
    if call == "route":
        return tuple(t.int() for t in _plain_route(s["experts"], s["n_experts"]))
    bounds, slots = s["bounds"], s["slots"]
    routed = bounds[-1]
    if call == "dispatch":
        out = torch.zeros((s["order"].numel(), s["tokens"].shape[1]), dtype=s["tokens"].dtype, device="cuda")
        out[:routed] = s["tokens"][s["order"][:routed] // slots]
        return out
    if call in ("dispatch_grad", "combine"):
        gathered = s["rows"][s["inverse"]].float()
        if call == "combine":
            gathered = gathered * s["weights"][:, :, None]
        return torch.where((s["inverse"] < routed)[:, :, None], gathered, 0.0).sum(1).to(s["rows"].dtype)
    if call == "combine_grad":
        grad, inside = s["tokens"].float(), s["inverse"] < routed
        grad_rows = torch.zeros_like(s["rows"])
        taken = s["order"][:routed]
        grad_rows[:routed] = (grad[taken // slots] * s["weights"].reshape(-1)[taken][:, None]).to(grad_rows.dtype)
        dots = (s["rows"][s["inverse"]].float() * grad[:, None, :]).sum(2)
        return grad_rows, torch.where(inside, dots, 0.0)
    x, w, trans = s["rows"], s["matrices"], s["op"] == "trans"
    if call == "product":
        out = torch.zeros((x.shape[0], w.shape[1 if trans else 2]), dtype=x.dtype, device="cuda")
        for e in range(s["n_experts"]):
            a, b = bounds[e], bounds[e + 1]
            if b > a:
                out[a:b] = x[a:b].float() @ (w[e].float().t() if trans else w[e].float())
        return out
    grad_rows, grad_w = torch.zeros_like(x), torch.zeros_like(w)
    for e in range(s["n_experts"]):
        a, b = bounds[e], bounds[e + 1]
        if b > a:
            g, xe, we = s["grad"][a:b].float(), x[a:b].float(), w[e].float()
            grad_rows[a:b] = g @ (we if trans else we.t())
            grad_w[e] = g.t() @ xe if trans else xe.t() @ g
    return grad_rows, grad_w


# -- reference -------------------------------------------------------------------------


def exact(case, seed):
    """The definitions in 64 bits, on the inputs as they are.  The places of a route are found by counting: the
    place of a slot is the number of slots with a smaller key plus the number of earlier ones with the same."""
    a, call = _operands(case, seed), case["call"]
    if call == "embedding":
        return a["values"][a["tokens"].long()].double() * case["scale"]
    if call == "embedding_grad":
        # rows in token order, summed in segments of equal tokens
        token, order = torch.sort(a["tokens"].long())
        out = torch.zeros((case["vocab"], case["width"]), dtype=torch.float64, device="cuda")
        present, lengths = torch.unique_consecutive(token, return_counts=True)
        step = max(1, (1 << 27) // case["tokens"])
        for c in range(0, case["width"], step):
            part = a["values"][:, c : c + step].double()[order] * case["scale"]
            out[present, c : c + step] = torch.segment_reduce(part, "sum", lengths=lengths, axis=0, unsafe=True)
        return out
    n_experts, experts = case["experts"], a["experts"].long()
    n, slots = experts.shape
    key = experts.reshape(-1)
    key = torch.where((key < 0) | (key >= n_experts), n_experts, key)
    inverse = torch.empty_like(key)
    offsets, start = [0], 0
    for e in range(n_experts + 1):
        mine = key == e
        inverse[mine] = torch.arange(start, start + int(mine.sum()), device="cuda")
        start += int(mine.sum())
        offsets.append(start)
    routed = offsets[n_experts]
    if call == "route":
        order = torch.empty_like(key)
        order[inverse] = torch.arange(n * slots, device="cuda")
        offsets = torch.tensor(offsets[:-1], dtype=torch.int32, device="cuda")
        return order.int(), inverse.int().reshape(n, slots), offsets
    rows = n * slots
    if call.startswith("product"):
        x, w, trans = a["rows"], a["matrices"], case["op"] == "trans"
        y = torch.zeros((rows, case["outer"]), dtype=torch.float64, device="cuda") if call == "product" else None
        gx = torch.zeros((rows, case["inner"]), dtype=torch.float64, device="cuda") if y is None else None
        gw = torch.zeros(w.shape, dtype=torch.float64, device="cuda") if y is None else None
        for e in range(n_experts):
            part = slice(offsets[e], offsets[e + 1])
            m = w[e].double()
            if y is not None:
                y[part] = x[part].double() @ (m.T if trans else m)
            else:
                d, v = a["grad"][part].double(), x[part].double()
                gx[part] = d @ (m if trans else m.T)
                gw[e] = d.T @ v if trans else v.T @ d
        return y if y is not None else (gx, gw)
    inverse = inverse.reshape(n, slots)
    inside = inverse < routed
    width = case["width"]
    if call == "dispatch":
        out = torch.zeros((rows, width), dtype=torch.float64, device="cuda")
        for j in range(slots):
            out[inverse[:, j][inside[:, j]]] = a["tokens"].double()[inside[:, j]]
        return out
    if call == "combine_grad":
        grad = a["tokens"].double()
        grad_rows = torch.zeros((rows, width), dtype=torch.float64, device="cuda")
        grad_w = torch.zeros((n, slots), dtype=torch.float64, device="cuda")
        for j in range(slots):
            at, here = inverse[:, j][inside[:, j]], inside[:, j]
            grad_rows[at] = grad[here] * a["weights"][here, j].double()[:, None]
            grad_w[here, j] = (grad[here] * a["rows"][at].double()).sum(1)
        return grad_rows, grad_w
    out = torch.zeros((n, width), dtype=torch.float64, device="cuda")
    for j in range(slots):
        here = inside[:, j]
        term = a["rows"][inverse[:, j][here]].double()
        if call == "combine":
            term = term * a["weights"][here, j].double()[:, None]
        out[here] += term
    return out
