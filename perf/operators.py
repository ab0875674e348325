"""The training operators around the encoded gradient path, as cases that can be timed and compared.

Three operators, in the forms a training program calls them:

  clip       the global L2 norm over a list of separately allocated gradient tensors of mixed types, and the
             clipped gradients (fp32 / bf16 leaves gathered into their bucket arenas, BFP8 by their scales)
  norm       root-mean-square norm of x + residual, its output in the codec's 8 bits with scales; and its gradient
  embedding  rows of a token table (fp32, bf16, or as it lies in BFP8) times a scale; and the table's gradient,
             summed over equal tokens in the order in which they occur

`own` False computes them from elementary torch operations, True through nntrain_b200.
"""
import math
import random

import torch

own = False

QWEN2_HIDDEN, QWEN2_LAYERS, QWEN2_KV, QWEN2_INTERMEDIATE, QWEN2_VOCAB = 1536, 28, 256, 8960, 151936
SMALL_WIDTH, SMALL_LAYERS, SMALL_FFN, SMALL_VOCAB = 512, 8, 2048, 32000
FLT_MIN = 1.1754943508222875e-38
EPSILON = 1e-6


def listed():
    return [
        # gradients of rank-8 adapters on the query and value projections: over a hundred small leaves, latency
        {"name": "clip_adapter_f32", "op": "clip", "list": "adapter", "types": "f32", "block": 0, "max_norm": 1.0},
        # a small decoder Transformer trained in bf16 with fp32 norm and bias gradients, into its two arenas
        {"name": "clip_small_mixed", "op": "clip", "list": "small", "types": "mixed", "block": 0, "max_norm": 1.0},
        # the same model after the compressed all-reduce: matrices in BFP8 (block 32), clipped by their scales
        {"name": "clip_small_bfp8", "op": "clip", "list": "small", "types": "bfp8", "block": 32, "max_norm": 1.0},
        # the benchmark's 338-tensor list of 1.54 G fp32 values, leaves gathered into one arena
        {"name": "clip_qwen2_f32", "op": "clip", "list": "qwen2", "types": "f32", "block": 0, "max_norm": 1.0},
        # one token of a generation step, encoded for an 8-bit product
        {"name": "norm_token_bf16", "op": "norm", "rows": 1, "width": 1536, "type": "bf16", "residual": True, "block": 32},
        # a training batch of eight sequences of 2048
        {"name": "norm_batch_bf16", "op": "norm", "rows": 16384, "width": 1536, "type": "bf16", "residual": True, "block": 32},
        # a ragged fp32 batch of an odd width, one scale a row
        {"name": "norm_odd_f32", "op": "norm", "rows": 3001, "width": 771, "type": "f32", "residual": True, "block": 0},
        # the gradient of a small ragged batch
        {"name": "norm_gradient_odd_f32", "op": "norm_gradient", "rows": 517, "width": 771, "type": "f32", "residual": True},
        # the gradient of a long training batch
        {"name": "norm_gradient_bf16", "op": "norm_gradient", "rows": 32768, "width": 1536, "type": "bf16", "residual": True},
        # a batch's rows out of the parameters as they are published, in BFP8
        {"name": "embedding_bfp8", "op": "embedding", "tokens": 8192, "vocab": QWEN2_VOCAB, "width": 1536, "table": "bfp8",
         "type": "bf16", "block": 32, "padded": 0.0},
        # the largest tensor of the 1.54 G arena: the whole table's gradient written, most rows zero
        {"name": "embedding_gradient_whole", "op": "embedding_gradient", "tokens": 8192, "vocab": QWEN2_VOCAB, "width": 1536,
         "type": "bf16", "table": "f32", "add": False, "padded": 0.0},
        # a later micro-batch of padded sequences, added to the gradient that is there
        {"name": "embedding_gradient_added", "op": "embedding_gradient", "tokens": 65536, "vocab": SMALL_VOCAB, "width": 512,
         "type": "f32", "table": "f32", "add": True, "padded": 0.1},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["clip", "clip", "norm", "norm_gradient", "embedding", "embedding_gradient"])
    if op == "clip":
        tensors = _log(rng, 1, 400)
        return {"op": op, "list": "drawn", "shape": rng.randrange(1 << 30), "tensors": tensors,
                "values": max(tensors, _log(rng, 1000, 600_000_000)), "types": rng.choice(["f32", "bf16", "mixed", "bfp8"]),
                "block": rng.choice([32, 128, 96, 0]), "max_norm": rng.choice([0.01, 1.0, 1e6])}
    if op in ("norm", "norm_gradient"):
        block = rng.choice([0, 32, 64, 128])
        width = _log(rng, 33, 9000)
        if block:
            width = max(block, width // block * block)
        case = {"op": op, "rows": max(1, min(_log(rng, 1, 65536), 60_000_000 // width)), "width": width,
                "type": rng.choice(["bf16", "f32"]), "residual": rng.random() < 0.7}
        return dict(case, block=block) if op == "norm" else case
    width = _log(rng, 33, 4200) if rng.random() < 0.4 else _log(rng, 2, 130) * 32
    tokens = max(1, min(_log(rng, 1, 131072), 120_000_000 // width))
    vocab = min(_log(rng, 100, 152_000), 230_000_000 // width)
    case = {"op": op, "tokens": tokens, "vocab": vocab, "width": width, "type": rng.choice(["bf16", "f32"]),
            "padded": rng.choice([0.0, 0.2])}
    if op == "embedding":
        return dict(case, table=rng.choice(["f32", "bf16", "bfp8"]), block=rng.choice([32, 128, 0]))
    return dict(case, table=rng.choice(["f32", "f32", "bf16"]), add=False) if rng.random() < 0.5 else dict(case, table="f32", add=True)


# ---- inputs ---------------------------------------------------------------------

def _numels(case):
    """(length, is a matrix) of the list's tensors."""
    if case["list"] == "adapter":
        layer = [8 * QWEN2_HIDDEN, QWEN2_HIDDEN * 8, 8 * QWEN2_HIDDEN, QWEN2_KV * 8]
        return [(n, True) for n in layer * QWEN2_LAYERS]
    if case["list"] == "small":
        w, f = SMALL_WIDTH, SMALL_FFN
        layer = [(3 * w * w, True), (3 * w, False), (w * w, True), (w, False), (w, False), (w, False), (w * f, True),
                 (f, False), (f * w, True), (w, False), (w, False), (w, False)]
        return [(SMALL_VOCAB * w, True)] + layer * SMALL_LAYERS + [(w, False), (w, False)]
    if case["list"] == "qwen2":
        h, kv, inter = QWEN2_HIDDEN, QWEN2_KV, QWEN2_INTERMEDIATE
        layer = [(h * h, True), (h, False), (h * kv, True), (kv, False), (h * kv, True), (kv, False), (h * h, True),
                 (h * inter, True), (h * inter, True), (inter * h, True), (h, False), (h, False)]
        return [(QWEN2_VOCAB * h, True)] + layer * QWEN2_LAYERS + [(h, False)]
    # drawn: lengths spread over their logarithm, odd ones among them, that add up to about case["values"]
    rng = random.Random(case["shape"])
    parts = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(case["tensors"])]
    lengths = [max(1, int(case["values"] * p / sum(parts))) for p in parts]
    return [(n, rng.random() < 0.6) for n in lengths]


def _types(case):
    """The type of each tensor of the list."""
    if case["types"] == "mixed":
        return ["bf16" if matrix else "f32" for _, matrix in _numels(case)]
    if case["types"] == "bfp8":
        return ["bfp8" if matrix else "f32" for _, matrix in _numels(case)]
    return [case["types"] for _ in _numels(case)]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _dtype(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _encode(x, block):
    """The codec's payload and scales of a flat fp32 tensor; block 0: one scale for all of it."""
    n = x.numel()
    block = n if block == 0 or block > n else block
    count = (n + block - 1) // block
    padded = torch.nn.functional.pad(x, (0, count * block - n)).view(count, block)
    maximum = padded.abs().amax(dim=1)
    scales = torch.where(maximum == 0, torch.ones_like(maximum), maximum / 127.0)
    codes = torch.clamp(torch.round(padded / scales[:, None]), -127, 127).to(torch.int8)
    return codes.view(-1)[:n].clone(), scales


def _decode(payload, scales, block):
    n = payload.numel()
    if block == 0 or block >= n:
        return payload.float() * scales
    return payload.float() * scales.repeat_interleave(block)[:n]


def _tokens(case, g):
    """Tokens by a law of about 1 / rank, as text has them; -1 where a sequence is padded."""
    u = torch.rand(case["tokens"], generator=g, device="cuda", dtype=torch.float64)
    tokens = (torch.exp(u * math.log(case["vocab"] + 1.0)) - 1.0).to(torch.int64).clamp_(0, case["vocab"] - 1)
    if case["padded"]:
        pad = torch.rand(case["tokens"], generator=g, device="cuda") < case["padded"]
        tokens = torch.where(pad, torch.full_like(tokens, -1), tokens)
    return tokens


def prepare(case, seed):
    g = _generator(seed)
    op, s = case["op"], {"case": case}

    def normal(*shape, sigma=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").mul_(sigma).to(dtype)

    if op == "clip":
        tensors, scales, types = [], [], _types(case)
        for (n, _), kind in zip(_numels(case), types):
            sigma = math.exp(math.log(1e-5) + torch.rand(1, generator=torch.Generator().manual_seed(seed + 31 * len(tensors))).item()
                             * math.log(1e3))
            x = normal(n, sigma=sigma, dtype=_dtype(kind))
            payload_scales = None
            if kind == "bfp8":
                x, payload_scales = _encode(x, case["block"])
            tensors.append(x)
            scales.append(payload_scales)
        # where the clipped gradients go: one arena for each type, tensors one after another in it
        arenas = {kind: torch.zeros(sum(t.numel() for t, k in zip(tensors, types) if k == kind), dtype=_dtype(kind), device="cuda")
                  for kind in ("f32", "bf16") if kind in types}
        if "bfp8" in types:
            arenas["bfp8"] = torch.zeros(sum(v.numel() for v in scales if v is not None), device="cuda")
        taken, destinations = {kind: 0 for kind in arenas}, []
        for t, v, kind in zip(tensors, scales, types):
            n = t.numel() if v is None else v.numel()
            destinations.append(arenas[kind][taken[kind]:taken[kind] + n])
            taken[kind] += n
        s |= {"tensors": tensors, "scales": scales, "types": types, "arenas": arenas, "destinations": destinations,
              "norm": torch.zeros(2, device="cuda"), "norms": torch.zeros(len(tensors), device="cuda")}
        if own:
            # the list of addresses and lengths that a program builds once for its leaves
            from nntrain_b200.native import GradientTensorList
            s["list"] = GradientTensorList(0, tensors, scales, [case["block"]] * len(tensors), destinations)
        return s
    if op in ("norm", "norm_gradient"):
        rows, width, dtype = case["rows"], case["width"], _dtype(case["type"])
        s["weight"] = 1.0 + normal(width, sigma=0.2)
        if op == "norm":
            s["x"] = normal(rows, width, dtype=dtype)
            s["residual"] = normal(rows, width, sigma=3.0, dtype=dtype) if case["residual"] else None
            blocks = rows if case["block"] == 0 else rows * (width // case["block"])
            s |= {"sum": torch.empty_like(s["x"]) if case["residual"] else None,
                  "y": torch.empty(rows, width, dtype=torch.bfloat16, device="cuda"),
                  "payload": torch.empty(rows, width, dtype=torch.int8, device="cuda"),
                  "scales": torch.empty(blocks, device="cuda"), "inverse": torch.empty(rows, device="cuda")}
            return s
        s["input"] = normal(rows, width, sigma=3.0, dtype=dtype)
        s["inverse"] = torch.rsqrt(s["input"].float().square().mean(dim=1) + EPSILON)
        s["y_gradient"] = normal(rows, width, sigma=1e-3, dtype=dtype)
        s["residual_gradient"] = normal(rows, width, sigma=1e-3, dtype=dtype) if case["residual"] else None
        s |= {"x_gradient": torch.empty_like(s["input"]), "weight_gradient": torch.empty(width, device="cuda")}
        return s
    width, vocab = case["width"], case["vocab"]
    s["tokens"] = _tokens(case, g)
    s["scale"] = math.sqrt(width)
    if op == "embedding":
        table = normal(vocab * width, sigma=0.02, dtype=_dtype(case["table"]))
        s["scales"] = None
        if case["table"] == "bfp8":
            table, s["scales"] = _encode(table, case["block"])
        s |= {"table": table.view(vocab, width), "out": torch.empty(case["tokens"], width, dtype=_dtype(case["type"]), device="cuda")}
        return s
    s["out_gradient"] = normal(case["tokens"], width, sigma=1e-3, dtype=_dtype(case["type"]))
    s["table_gradient"] = normal(vocab, width, sigma=1e-3, dtype=_dtype(case["table"]))
    return s


# ---- one pass -------------------------------------------------------------------

def _clip(s):
    case = s["case"]
    if own:
        from nntrain_b200.native import GradientNorm
        GradientNorm.clip_tensors(0, s["list"], case["max_norm"], s["norm"], tensor_norms=s["norms"])
        return {"norm": s["norm"], "norms": s["norms"], "arenas": s["arenas"]}
    values = [t.float() if v is None else _decode(t, v, case["block"]) for t, v in zip(s["tensors"], s["scales"])]
    squares = torch.stack([v.square().sum(dtype=torch.float64) for v in values])
    norm = squares.sum().sqrt().float()
    coefficient = torch.where(norm > case["max_norm"], case["max_norm"] / (norm + 1e-6), torch.ones_like(norm))
    arenas = {}
    for kind in s["arenas"]:
        parts = [t if v is None else v for t, v, k in zip(s["tensors"], s["scales"], s["types"]) if k == kind]
        clipped = torch.cat(parts).float() * coefficient
        if kind == "bfp8":
            clipped = torch.where(coefficient == 1.0, clipped, clipped.clamp_min(FLT_MIN))
        arenas[kind] = clipped.to(_dtype(kind))
    return {"norm": torch.stack([norm, coefficient]), "norms": squares.sqrt().float(), "arenas": arenas}


def _norm(s):
    case = s["case"]
    if own:
        from nntrain_b200.native import RmsNorm
        RmsNorm.forward(0, s["x"], s["weight"], EPSILON, residual=s["residual"], residual_out=s["sum"], y=s["y"],
                        payload=s["payload"], scales=s["scales"], block_size=case["block"], inverse_rms=s["inverse"])
        return {"sum": s["sum"], "y": s["y"], "scales": s["scales"], "inverse": s["inverse"]}
    rows, width = case["rows"], case["width"]
    h = s["x"].float() if s["residual"] is None else s["x"].float() + s["residual"].float()
    inverse = 1.0 / torch.sqrt(h.square().mean(dim=1) + EPSILON)
    y = (h * inverse[:, None] * s["weight"]).view(-1, width if case["block"] == 0 else case["block"])
    maximum = y.abs().amax(dim=1)
    scales = torch.where(maximum == 0, torch.ones_like(maximum), maximum / 127.0)
    codes = torch.clamp(torch.round(y / scales[:, None]), -127, 127)
    # the 8-bit values, as the bf16 values that they stand for
    values = (codes * scales[:, None]).view(rows, width).to(torch.bfloat16)
    return {"sum": h.to(s["x"].dtype) if s["residual"] is not None else None, "y": values, "scales": scales, "inverse": inverse}


def _norm_gradient(s):
    if own:
        from nntrain_b200.native import RmsNorm
        RmsNorm.backward(0, s["y_gradient"], s["input"], s["weight"], s["inverse"], s["x_gradient"], s["weight_gradient"],
                         residual_gradient=s["residual_gradient"])
        return {"x": s["x_gradient"], "weight": s["weight_gradient"]}
    dy, h, inverse = s["y_gradient"].float(), s["input"].float(), s["inverse"][:, None]
    normalized = h * inverse
    g = dy * s["weight"]
    dx = inverse * (g - normalized * (g * normalized).mean(dim=1, keepdim=True))
    if s["residual_gradient"] is not None:
        dx = dx + s["residual_gradient"].float()
    return {"x": dx.to(s["input"].dtype), "weight": (dy * normalized).sum(dim=0, dtype=torch.float64).float()}


def _embedding(s):
    case = s["case"]
    if own:
        from nntrain_b200.native import TokenEmbedding
        TokenEmbedding.lookup(0, s["tokens"], s["table"], s["out"], scale=s["scale"], table_scales=s["scales"],
                              block_size=case["block"])
        return {"out": s["out"]}
    tokens = s["tokens"].clamp_min(0)
    rows = s["table"][tokens].float()
    if s["scales"] is not None:
        values = case["vocab"] * case["width"]
        block = values if case["block"] == 0 else case["block"]
        places = tokens[:, None] * case["width"] + torch.arange(case["width"], device="cuda")
        rows = rows * s["scales"][places // block]
    out = torch.where((s["tokens"] >= 0)[:, None], rows * s["scale"], torch.zeros_like(rows))
    return {"out": out.to(s["out"].dtype)}


def _embedding_gradient(s):
    case = s["case"]
    if own:
        from nntrain_b200.native import TokenEmbedding
        TokenEmbedding.gradient(0, s["tokens"], s["out_gradient"], s["table_gradient"], scale=s["scale"], accumulate=case["add"])
        return {"table": s["table_gradient"]}
    valid = (s["tokens"] >= 0)[:, None]
    rows = s["out_gradient"].float() * s["scale"]
    rows = torch.where(valid, rows, torch.zeros_like(rows))
    tokens = s["tokens"].clamp_min(0)
    if case["add"]:
        return {"table": s["table_gradient"].index_add_(0, tokens, rows)}
    total = torch.zeros(case["vocab"], case["width"], device="cuda").index_add_(0, tokens, rows)
    return {"table": total.to(s["table_gradient"].dtype)}


def run(state):
    return {"clip": _clip, "norm": _norm, "norm_gradient": _norm_gradient, "embedding": _embedding,
            "embedding_gradient": _embedding_gradient}[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------

def _size(name):
    return 2 if name == "bf16" else 4


def work(case):
    op = case["op"]
    if op == "clip":
        moved = flops = 0
        for (n, _), kind in zip(_numels(case), _types(case)):
            if kind == "bfp8":
                scales = 1 if case["block"] == 0 else -(-n // case["block"])
                moved += n + 8 * scales                      # payload and scales read, scales written
            else:
                moved += 2 * n * _size(kind)                 # read and written once
            flops += 3 * n
        return {"bytes": moved, "flops": flops}
    if op in ("norm", "norm_gradient"):
        n, size = case["rows"] * case["width"], _size(case["type"])
        if op == "norm":
            blocks = case["rows"] if case["block"] == 0 else n // case["block"]
            moved = n * size * (3 if case["residual"] else 1) + n * 3 + 4 * blocks + 4 * case["rows"] + 4 * case["width"]
            return {"bytes": moved, "flops": 8 * n}
        return {"bytes": n * size * (4 if case["residual"] else 3) + 4 * case["rows"] + 8 * case["width"], "flops": 10 * n}
    # different rows among the tokens, by the law of _tokens: those named once a pass or more, and some of the others
    tokens, vocab, width = case["tokens"], case["vocab"], case["width"]
    often = min(vocab, max(1.0, tokens / math.log(vocab + 1.0)))
    different = min(tokens, vocab, int(often * (1.0 + math.log(vocab / often))))
    if op == "embedding":
        size = {"f32": 4.0, "bf16": 2.0, "bfp8": 1.0 + (4.0 / case["block"] if case["block"] else 0.0)}[case["table"]]
        return {"bytes": 8 * tokens + different * width * size + tokens * width * _size(case["type"]), "flops": tokens * width}
    written = 2 * different if case["add"] else vocab
    return {"bytes": 8 * tokens + tokens * width * _size(case["type"]) + written * width * _size(case["table"]),
            "flops": 2 * tokens * width}


# ---- the definition in 64 bits ----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "clip":
        def values(i):
            t, v = s["tensors"][i], s["scales"][i]
            if v is None:
                return t.double()
            if v.numel() == 1:
                return t.double() * v.double()
            place = torch.arange(t.numel(), device="cuda").div_(case["block"], rounding_mode="floor")
            return t.double() * v.double()[place]

        norms = [float(torch.linalg.vector_norm(values(i))) for i in range(len(s["tensors"]))]
        norm = math.sqrt(math.fsum(v * v for v in norms))
        c = case["max_norm"] / (norm + 1e-6) if norm > case["max_norm"] else 1.0
        arenas = {kind: torch.empty(a.numel(), dtype=torch.float64, device="cuda") for kind, a in s["arenas"].items()}
        taken = {kind: 0 for kind in arenas}
        for t, v, kind in zip(s["tensors"], s["scales"], s["types"]):
            part = (t if v is None else v).double() * c
            if v is not None and c != 1.0:
                part = part.clamp_min(FLT_MIN)
            arenas[kind][taken[kind]:taken[kind] + part.numel()] = part
            taken[kind] += part.numel()
        return {"norm": torch.tensor([norm, c], dtype=torch.float64), "norms": torch.tensor(norms, dtype=torch.float64), "arenas": arenas}
    if op == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h += s["residual"].double()
        inverse = (torch.einsum("rc,rc->r", h, h) / case["width"] + EPSILON).pow(-0.5)
        y = torch.einsum("rc,r,c->rc", h, inverse, s["weight"].double())
        blocks = y.reshape(s["scales"].numel(), -1)
        low, high = blocks.aminmax(dim=1)
        largest = torch.maximum(-low, high)
        scales = largest / 127.0
        scales[largest == 0] = 1.0
        codes = (blocks / scales.unsqueeze(1)).round_().clamp_(-127, 127)
        return {"sum": h if s["residual"] is not None else None, "y": (codes * scales.unsqueeze(1)).reshape(y.shape),
                "scales": scales, "inverse": inverse}
    if op == "norm_gradient":
        h, dy, w, r = s["input"].double(), s["y_gradient"].double(), s["weight"].double(), s["inverse"].double()
        along = torch.einsum("rc,rc,c->r", dy, h, w) * r.pow(3) / case["width"]
        dx = torch.einsum("rc,c,r->rc", dy, w, r) - h * along.unsqueeze(1)
        if s["residual_gradient"] is not None:
            dx += s["residual_gradient"].double()
        return {"x": dx, "weight": torch.einsum("rc,rc,r->c", dy, h, r)}
    valid = s["tokens"] >= 0
    if op == "embedding":
        out = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
        named = s["tokens"][valid]
        rows = s["table"][named].double()
        if s["scales"] is not None:
            if case["block"] == 0:
                rows *= s["scales"].double()
            else:
                first = named * case["width"]
                column = torch.arange(case["width"], device="cuda")
                rows *= s["scales"].double()[torch.div(first.unsqueeze(1) + column, case["block"], rounding_mode="floor")]
        out[valid] = rows * s["scale"]
        return {"out": out}
    table = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device="cuda")
    table.index_add_(0, s["tokens"][valid], s["out_gradient"][valid].double(), alpha=s["scale"])
    if case["add"]:
        table += s["table_gradient"].double()
    return {"table": table}
