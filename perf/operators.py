"""The operators of the training and serving side of the embedding -> norm -> rotation path, as cases to be measured.

Five calls: the scaled embedding lookup, the gradient of the table, the head norms of queries and keys with the
rotation in the same pass, their gradient, and the gradient of the RMS norm.  Each has a plain form in elementary
torch operations (f32 inside, one rounding at the end) and the package's own call; ``exact`` states the definition
again in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ID_DTYPES = {"u32": torch.uint32, "i32": torch.int32, "i64": torch.int64}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
ZIPF = 1.1


def listed():
    return [
        # one decoding step of 64 sequences: 64 rows out of a large table, where the launch is the time
        {"name": "lookup-decode-bf16", "op": "lookup", "dtype": "bf16", "vocab": 128256, "hidden": 4096, "tokens": 64,
         "ids": "zipf", "id_dtype": "u32"},
        # the prompt of 8 x 512 tokens of the f32 embedding configuration
        {"name": "lookup-prompt-f32", "op": "lookup", "dtype": "f32", "vocab": 32000, "hidden": 4096, "tokens": 4096,
         "ids": "uniform", "id_dtype": "i64"},
        # a training step of 32 x 2048 tokens with text's skew (the hottest id has thousands of tokens): a fresh
        # dense gradient of the large table
        {"name": "table-grad-zipf-bf16", "op": "table_grad", "dtype": "bf16", "out": "bf16", "accumulate": False,
         "vocab": 128256, "hidden": 4096, "tokens": 65536, "ids": "zipf", "id_dtype": "u32"},
        # a micro-batch added to the f32 gradient that the optimizer reads: only the rows that occur are touched
        {"name": "table-grad-accumulate-f32", "op": "table_grad", "dtype": "bf16", "out": "f32", "accumulate": True,
         "vocab": 32000, "hidden": 4096, "tokens": 4096, "ids": "uniform", "id_dtype": "i64"},
        # a short ragged batch over a small model's table, f16
        {"name": "table-grad-ragged-f16", "op": "table_grad", "dtype": "f16", "out": "f16", "accumulate": False,
         "vocab": 50021, "hidden": 1000, "tokens": 3001, "ids": "zipf", "id_dtype": "i64"},
        # one decoding step of 64 sequences at their own positions, q and k as views of the packed projection
        {"name": "rotate-decode-bf16", "op": "rotate", "dtype": "bf16", "table_dtype": "bf16", "batch": 64, "length": 1,
         "q_heads": 32, "k_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "positions": True},
        # a prompt batch with grouped key heads
        {"name": "rotate-prompt-bf16", "op": "rotate", "dtype": "bf16", "table_dtype": "bf16", "batch": 8, "length": 2048,
         "q_heads": 32, "k_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "positions": False},
        # adjacent pairs, a part of each head rotated, odd lengths, f16 with f32 angles
        {"name": "rotate-partial-f16", "op": "rotate", "dtype": "f16", "table_dtype": "f32", "batch": 3, "length": 1021,
         "q_heads": 12, "k_heads": 12, "dim": 80, "rotary": 32, "interleaved": True, "positions": True},
        # the gradient in a training step of long sequences
        {"name": "rotate-grad-bf16", "op": "rotate_grad", "dtype": "bf16", "table_dtype": "f32", "batch": 4, "length": 4096,
         "q_heads": 32, "k_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "positions": False},
        # a small ragged one in f32
        {"name": "rotate-grad-f32", "op": "rotate_grad", "dtype": "f32", "table_dtype": "f32", "batch": 1, "length": 777,
         "q_heads": 16, "k_heads": 2, "dim": 64, "rotary": 64, "interleaved": False, "positions": True},
        # the large residual norm configuration, trained: the residual stream's gradient is added in the same pass
        {"name": "norm-grad-bf16", "op": "norm_grad", "dtype": "bf16", "rows": 65536, "cols": 8192, "residual": True},
        # few rows in f32
        {"name": "norm-grad-f32", "op": "norm_grad", "dtype": "f32", "rows": 509, "cols": 4096, "residual": False},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["lookup", "table_grad", "rotate", "rotate_grad", "norm_grad"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("lookup", "table_grad"):
        hidden = _log(rng, 64, 8192)
        if rng.random() < 0.75:
            hidden = (hidden + 63) // 64 * 64
        vocab = _log(rng, 1000, min(160000, (1 << 30) // (hidden * BYTES[dtype])))
        c = {"op": op, "dtype": dtype, "vocab": vocab, "hidden": hidden, "tokens": _log(rng, 1, 65536),
             "ids": rng.choice(["uniform", "zipf"]), "id_dtype": rng.choice(["u32", "i32", "i64"])}
        if op == "table_grad":
            c["out"] = rng.choice([dtype, "f32"])
            c["accumulate"] = rng.random() < 0.4
        return c
    if op == "norm_grad":
        cols = _log(rng, 256, 8192)
        if rng.random() < 0.75:
            cols = (cols + 63) // 64 * 64
        rows = _log(rng, 1, (1 << 28) // cols)
        return {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "residual": rng.random() < 0.5}
    dim = rng.choice([32, 64, 72, 80, 96, 128, 128, 192, 256])
    k_heads = rng.choice([1, 2, 4, 8])
    length = _log(rng, 1, 8192) if rng.random() < 0.8 else 1
    return {"op": op, "dtype": dtype, "table_dtype": rng.choice([dtype, "f32"]), "batch": _log(rng, 1, max(1, 16384 // length)),
            "length": length, "q_heads": k_heads * rng.choice([1, 2, 4]), "k_heads": k_heads, "dim": dim,
            "rotary": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.4,
            "positions": rng.random() < 0.6}


def _ids(case, gen):
    """Token ids: uniform over the vocabulary, or rank k with probability ~ k^-1.1 (rank k is id k - 1)."""
    n, vocab = case["tokens"], case["vocab"]
    if case["ids"] == "uniform":
        ids = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
    else:
        p = torch.arange(1, vocab + 1, device="cuda", dtype=torch.float64).pow(-ZIPF)
        u = torch.rand(n, device="cuda", dtype=torch.float64, generator=gen)
        cdf = p.cumsum(0)
        ids = torch.searchsorted(cdf, u * cdf[-1]).clamp_(max=vocab - 1)
    if case["id_dtype"] == "u32":
        return ids.to(torch.int32).view(torch.uint32)
    return ids.to(ID_DTYPES[case["id_dtype"]])


def _normal(shape, dtype, gen, mean=0.0, std=1.0):
    return torch.randn(shape, device="cuda", dtype=dtype, generator=gen).mul_(std).add_(mean)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case, "status": torch.zeros(4, dtype=torch.int64, device="cuda")}
    if case["op"] in ("lookup", "table_grad"):
        state["ids"] = _ids(case, gen)
        state["scale"] = math.sqrt(case["hidden"])
        if case["op"] == "lookup":
            state["table"] = _normal((case["vocab"], case["hidden"]), dtype, gen, std=0.02)
        else:
            state["grad"] = _normal((case["tokens"], case["hidden"]), dtype, gen, std=0.01)
            if case["accumulate"]:  # the sum of the micro-batches before this one
                state["sum"] = _normal((case["vocab"], case["hidden"]), DTYPES[case["out"]], gen, std=0.1)
        return state
    if case["op"] == "norm_grad":
        shape = (case["rows"], case["cols"])
        state["x"] = _normal(shape, dtype, gen)
        state["grad"] = _normal(shape, dtype, gen, std=0.01)
        state["weight"] = _normal(shape[1:], dtype, gen, mean=1.0, std=0.1)
        state["residual_grad"] = _normal(shape, dtype, gen, std=0.01) if case["residual"] else None
        return state
    b, t, hq, hk, d, rd = (case[k] for k in ("batch", "length", "q_heads", "k_heads", "dim", "rotary"))
    # q, k and v leave the projection packed: the heads are views of its rows
    qkv = _normal((b, t, hq + 2 * hk, d), dtype, gen)
    state["q"], state["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    state["q_weight"] = _normal((d,), dtype, gen, mean=1.0, std=0.1)
    state["k_weight"] = _normal((d,), dtype, gen, mean=1.0, std=0.1)
    longest = t + 4096 if case["positions"] else t
    freq = 10000.0 ** (-torch.arange(0, rd, 2, device="cuda", dtype=torch.float64) / rd)
    angle = torch.arange(longest, device="cuda", dtype=torch.float64)[:, None] * freq
    state["cos"], state["sin"] = angle.cos().to(DTYPES[case["table_dtype"]]), angle.sin().to(DTYPES[case["table_dtype"]])
    state["positions"] = None
    if case["positions"]:  # each sequence goes on from where its cache ends
        start = torch.randint(0, 4097, (b, 1), device="cuda", generator=gen)
        state["positions"] = (start + torch.arange(t, device="cuda")).contiguous()
    if case["op"] == "rotate_grad":
        state["grad_q"] = _normal((b, t, hq, d), dtype, gen, std=0.01)
        state["grad_k"] = _normal((b, t, hk, d), dtype, gen, std=0.01)
    return state


# ---- plain forms -----------------------------------------------------------------------------


def _long(ids):
    return (ids.view(torch.int32) if ids.dtype == torch.uint32 else ids).long()


def _plain_lookup(s):
    table = s["table"]
    return (table[_long(s["ids"])].float() * s["scale"]).to(table.dtype)


def _plain_table_grad(s):
    case, grad = s["case"], s["grad"]
    terms = grad.float() * s["scale"]
    out = DTYPES[case["out"]]
    if not case["accumulate"]:
        total = torch.zeros(case["vocab"], case["hidden"], dtype=torch.float32, device=grad.device)
        return total.index_add_(0, _long(s["ids"]), terms).to(out)
    if out == torch.float32:
        return s["sum"].index_add_(0, _long(s["ids"]), terms)
    return s["sum"].copy_(s["sum"].float().index_add_(0, _long(s["ids"]), terms))


def _turn(x, cos, sin, interleaved, back=False):
    """The first 2 * cos.shape[-1] columns of x rotated by the angle (by its opposite with `back`)."""
    half = cos.shape[-1]
    sin = -sin if back else sin
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _angles(s, t):
    cos, sin = s["cos"].float(), s["sin"].float()
    if s["positions"] is None:
        return cos[:t, None], sin[:t, None]
    return cos[s["positions"]][:, :, None], sin[s["positions"]][:, :, None]


def _plain_heads(x, weight, cos, sin, interleaved):
    f = x.float()
    r = torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
    return _turn(f * r * weight.float(), cos, sin, interleaved).to(x.dtype)


def _plain_heads_grad(grad, x, weight, cos, sin, interleaved):
    f = x.float()
    r = torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
    unit = f * r
    v = _turn(grad.float(), cos, sin, interleaved, back=True)
    scaled = v * weight.float()
    dx = r * (scaled - unit * (scaled * unit).mean(-1, keepdim=True))
    return dx.to(x.dtype), (v * unit).sum((0, 1, 2))


def _plain_norm_grad(s):
    x, grad = s["x"].float(), s["grad"].float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    unit = x * r
    scaled = grad * s["weight"].float()
    dx = r * (scaled - unit * (scaled * unit).mean(-1, keepdim=True))
    if s["residual_grad"] is not None:
        dx = dx + s["residual_grad"].float()
    return dx.to(s["x"].dtype), (grad * unit).sum(0)


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        import candle_b200 as cb

        if op == "lookup":
            return cb.embedding_scaled(s["table"], s["ids"], s["scale"], check=False, status=s["status"])
        if op == "table_grad":
            return cb.embedding_backward(s["grad"], s["ids"], case["vocab"], scale=s["scale"], out=s.get("sum"),
                                         accumulate=case["accumulate"], out_dtype=DTYPES[case["out"]], check=False,
                                         status=s["status"])
        if op == "norm_grad":
            return cb.rms_norm_backward(s["grad"], s["x"], s["weight"], EPS, grad_sum=s["residual_grad"])
        if op == "rotate":
            return cb.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], EPS, s["cos"], s["sin"],
                                   positions=s["positions"], interleaved=case["interleaved"], check=False,
                                   status=s["status"])
        return cb.qk_norm_rope_backward(s["grad_q"], s["grad_k"], s["q"], s["k"], s["q_weight"], s["k_weight"], EPS,
                                        s["cos"], s["sin"], positions=s["positions"], interleaved=case["interleaved"],
                                        check=False, status=s["status"])
    if op == "lookup":
        return _plain_lookup(s)
    if op == "table_grad":
        return _plain_table_grad(s)
    if op == "norm_grad":
        return _plain_norm_grad(s)
    cos, sin = _angles(s, case["length"])
    inter = case["interleaved"]
    if op == "rotate":
        return (_plain_heads(s["q"], s["q_weight"], cos, sin, inter),
                _plain_heads(s["k"], s["k_weight"], cos, sin, inter))
    dq, dwq = _plain_heads_grad(s["grad_q"], s["q"], s["q_weight"], cos, sin, inter)
    dk, dwk = _plain_heads_grad(s["grad_k"], s["k"], s["k_weight"], cos, sin, inter)
    return dq, dk, dwq, dwk


# ---- work ------------------------------------------------------------------------------------


def _distinct(case):
    """The expected number of different ids among the case's tokens."""
    n, vocab = case["tokens"], case["vocab"]
    if case["ids"] == "uniform":
        return vocab * -math.expm1(n * math.log1p(-1.0 / vocab))
    p = torch.arange(1, vocab + 1, dtype=torch.float64).pow(-ZIPF)
    return float(-torch.expm1(n * torch.log1p(-p / p.sum())).sum())


def work(case):
    op, size = case["op"], BYTES[case["dtype"]]
    if op in ("lookup", "table_grad"):
        n, hidden = case["tokens"], case["hidden"]
        ids = n * {"u32": 4, "i32": 4, "i64": 8}[case["id_dtype"]]
        if op == "lookup":
            return {"bytes": ids + (_distinct(case) + n) * hidden * size, "flops": n * hidden}
        out = BYTES[case["out"]]
        written = 2 * _distinct(case) if case["accumulate"] else case["vocab"]
        return {"bytes": ids + n * hidden * size + written * hidden * out, "flops": 2 * n * hidden}
    if op == "norm_grad":
        e = case["rows"] * case["cols"]
        return {"bytes": e * size * (4 if case["residual"] else 3) + case["cols"] * (size + 4), "flops": 10 * e}
    tokens, d = case["batch"] * case["length"], case["dim"]
    e = tokens * (case["q_heads"] + case["k_heads"]) * d
    rows = tokens if case["positions"] else case["length"]
    angles = rows * case["rotary"] * BYTES[case["table_dtype"]] + (8 * tokens if case["positions"] else 0)
    if op == "rotate":
        return {"bytes": 2 * e * size + 2 * d * size + angles, "flops": 7 * e}
    return {"bytes": 3 * e * size + 2 * d * (size + 4) + angles, "flops": 14 * e}


# ---- the definitions in 64 bits --------------------------------------------------------------


def _exact_rotation(case, s):
    """Per (sequence, token): the rotation as a complex factor for each pair."""
    at = s["positions"]
    if at is None:
        at = torch.arange(case["length"], device="cuda").expand(case["batch"], -1)
    return torch.complex(s["cos"].double(), s["sin"].double())[at].unsqueeze(2)


def _exact_pairs(x, rotary, interleaved):
    p = x[..., :rotary]
    if interleaved:
        return torch.view_as_complex(p.reshape(*p.shape[:-1], rotary // 2, 2).contiguous())
    return torch.complex(p[..., :rotary // 2].contiguous(), p[..., rotary // 2:].contiguous())


def _exact_unpairs(z, x, rotary, interleaved):
    y = x.clone()
    if interleaved:
        y[..., 0:rotary:2], y[..., 1:rotary:2] = z.real, z.imag
    else:
        y[..., :rotary // 2], y[..., rotary // 2:rotary] = z.real, z.imag
    return y


def _exact_norm_grad(g, x, w):
    """d/dx and d/dw of sum(g * x w / sqrt(mean(x^2) + eps)), row by row."""
    n = x.shape[-1]
    m = (x * x).sum(-1, keepdim=True) / n + EPS
    along = (g * w * x).sum(-1, keepdim=True)
    return g * w / m.sqrt() - x * along / (n * m * m.sqrt()), g * x / m.sqrt()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        return s["table"].double().mul(s["scale"]).index_select(0, _long(s["ids"]))
    if op == "table_grad":
        # sums of runs of equal ids in sorted order, as differences of running totals in 64 bits over a few columns at a time
        ids, perm = torch.sort(_long(s["ids"]), stable=True)
        last = torch.cat([ids[1:] != ids[:-1], ids.new_ones(1, dtype=torch.bool)]).nonzero()[:, 0]
        out = torch.zeros(case["vocab"], case["hidden"], dtype=torch.float64, device="cuda")
        for c in range(0, case["hidden"], 512):
            run_total = s["grad"][:, c:c + 512].double()[perm].cumsum(0)[last]
            out[ids[last], c:c + 512] = torch.diff(run_total, dim=0, prepend=torch.zeros_like(run_total[:1])) * s["scale"]
        return out.add_(s["sum"].double()) if case["accumulate"] else out
    if op == "norm_grad":
        dx = torch.empty(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
        dw = torch.zeros(case["cols"], dtype=torch.float64, device="cuda")
        for r in range(0, case["rows"], 8192):
            block = slice(r, r + 8192)
            dx[block], terms = _exact_norm_grad(s["grad"][block].double(), s["x"][block].double(), s["weight"].double())
            dw += terms.sum(0)
            if s["residual_grad"] is not None:
                dx[block] += s["residual_grad"][block].double()
        return dx, dw
    turn, rd, inter = _exact_rotation(case, s), case["rotary"], case["interleaved"]
    if op == "rotate":
        outs = []
        for x, w in ((s["q"].double(), s["q_weight"].double()), (s["k"].double(), s["k_weight"].double())):
            u = w * x / ((x * x).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt()
            outs.append(_exact_unpairs(_exact_pairs(u, rd, inter) * turn, u, rd, inter))
        return tuple(outs)
    dxs, dws = [], []
    for g, x, w in ((s["grad_q"].double(), s["q"].double(), s["q_weight"].double()),
                    (s["grad_k"].double(), s["k"].double(), s["k_weight"].double())):
        v = _exact_unpairs(_exact_pairs(g, rd, inter) * turn.conj(), g, rd, inter)
        dx, terms = _exact_norm_grad(v, x, w)
        dxs.append(dx)
        dws.append(terms.sum((0, 1, 2)))
    return (*dxs, *dws)
