"""What is measured of the sequence-model operators: token embeddings and their gradient, the root-mean-square norm on
a residual stream (with its gradient, and with 8-bit rows as its result), the gated linear recurrence over packed
sequences (with its gradient, and one token at a time) and products with 4-bit weights.

`run` computes one pass, in elementary torch operations or, where `own` is set, by the framework's kernels."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f64": torch.float64}
EPS = 1e-5


def listed():
    return [
        # a decoding step's tokens: latency
        {"name": "embed_fwd_decode", "op": "embed_fwd", "type": "f32", "tokens": 16, "vocab": 32768, "width": 2048},
        # a training batch's tokens: the copy rate
        {"name": "embed_fwd_batch", "op": "embed_fwd", "type": "f32", "tokens": 16384, "vocab": 65536, "width": 2048},
        # its gradient: frequent tokens, rows nobody asked for, a width that is no power of two
        {"name": "embed_bwd_batch", "op": "embed_bwd", "type": "f32", "tokens": 32768, "vocab": 50000, "width": 1000},
        # a small vocabulary, few tokens, rows without 16-byte alignment
        {"name": "embed_bwd_small_f64", "op": "embed_bwd", "type": "f64", "tokens": 2048, "vocab": 8192, "width": 513},
        # the norm between two layers in training: residual added, both kept
        {"name": "norm_fwd_batch", "op": "norm_fwd", "type": "f32", "rows": 16384, "cols": 4096},
        {"name": "norm_bwd_batch", "op": "norm_bwd", "type": "f32", "rows": 8192, "cols": 2560},
        # a batch of equal sequences
        {"name": "scan_fwd_batch", "op": "scan_fwd", "type": "f32", "tokens": 32768, "seqs": 8, "channels": 2048, "ragged": False},
        # packed sequences of uneven lengths
        {"name": "scan_bwd_ragged", "op": "scan_bwd", "type": "f32", "tokens": 32768, "seqs": 5, "channels": 1024, "ragged": True},
        # one long sequence, few channels: parallel over time or not at all
        {"name": "scan_fwd_long_f64", "op": "scan_fwd", "type": "f64", "tokens": 100001, "seqs": 1, "channels": 96, "ragged": False},
        # a decoding step: one token of each of 64 sequences
        {"name": "scan_step", "op": "scan_fwd", "type": "f32", "tokens": 64, "seqs": 64, "channels": 4096, "ragged": False},
        # a decoding step's largest product, one sequence
        {"name": "q4_one_row", "op": "q4", "rows": 1, "cols": 4096, "outs": 8192, "group": 128},
        # the norm with 8-bit rows and the product that reads them, 16 sequences
        {"name": "norm_q8_q4", "op": "norm_q8_q4", "rows": 16, "cols": 4096, "outs": 8192, "group": 64},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed_fwd", "embed_bwd", "norm_fwd", "norm_bwd", "scan_fwd", "scan_bwd", "step", "q4", "norm_q8_q4"])
    t = rng.choice(["f32", "f32", "f64"])
    most = (1 << 26) if t == "f32" else (1 << 25)  # values of the largest tensor: the largest listed case's
    if op in ("embed_fwd", "embed_bwd"):
        width = _spread(rng, 64, 4096)
        return {"op": op, "type": t, "tokens": min(_spread(rng, 1, 65536), most // (2 * width)),
                "vocab": min(_spread(rng, 256, 131072), most // width), "width": width}
    if op in ("norm_fwd", "norm_bwd"):
        cols = _spread(rng, 64, 16384)
        return {"op": op, "type": t, "rows": min(_spread(rng, 1, 32768), most // (2 * cols)), "cols": cols}
    if op == "step":
        seqs = _spread(rng, 1, 512)
        return {"op": "scan_fwd", "type": t, "tokens": seqs, "seqs": seqs, "channels": _spread(rng, 64, 8192), "ragged": False}
    if op in ("scan_fwd", "scan_bwd"):
        channels = _spread(rng, 64, 4096)
        tokens = min(_spread(rng, 64, 131072), most // (2 * channels))
        ragged = rng.random() < 0.5
        seqs = min(_spread(rng, 1, 64), tokens)
        return {"op": op, "type": t, "tokens": tokens if ragged else tokens // seqs * seqs, "seqs": seqs, "channels": channels,
                "ragged": ragged}
    group = rng.choice([32, 64, 128, 256])
    cols = max(group, _spread(rng, 512, 16384) // group * group) if rng.random() < 0.7 else _spread(rng, 512, 16384)
    return {"op": op, "rows": _spread(rng, 1, 32), "cols": cols, "outs": _spread(rng, 64, 16384), "group": group}


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _token_ids(n, vocab, g):
    """Token frequencies fall off as one over the rank."""
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    return ((vocab + 1.0) ** u - 1.0).long().clamp_(0, vocab - 1)


def _starts(case, seed):
    """Where each packed sequence begins, and the end: uneven lengths, an empty sequence now and then."""
    n, s = case["tokens"], case["seqs"]
    if not case["ragged"]:
        return [i * (n // s) for i in range(s + 1)]
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, n + 1, (s - 1,), generator=g).sort().values.tolist()
    return [0] + cuts + [n]


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    t = TYPES[case.get("type", "f32")]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device=DEV, dtype=t).mul_(std).add_(mean)

    s = {"case": dict(case), "op": op}
    if op in ("embed_fwd", "embed_bwd"):
        n, v, w = case["tokens"], case["vocab"], case["width"]
        s["ids"], s["scale"] = _token_ids(n, v, g), math.sqrt(w)
        if op == "embed_fwd":
            s["table"], s["res"] = normal(v, w, std=0.02), torch.empty(n, w, device=DEV, dtype=t)
        else:
            s["d_out"], s["d_table"] = normal(n, w, std=1e-3), torch.empty(v, w, device=DEV, dtype=t)
    elif op in ("norm_fwd", "norm_bwd"):
        r, c = case["rows"], case["cols"]
        s["gamma"] = normal(1, c, std=0.1, mean=1.0)
        s["x"], s["y"], s["inv"] = normal(r, c, std=2.0), torch.empty(r, c, device=DEV, dtype=t), torch.empty(r, 1, device=DEV, dtype=t)
        if op == "norm_fwd":
            s["residual"], s["h"] = normal(r, c, std=2.0), torch.empty(r, c, device=DEV, dtype=t)
        else:  # x is the kept sum, inv what the forward pass gave, d_sum the gradient that comes down the residual stream
            s["inv"] = (s["x"].double().square().mean(1, keepdim=True) + EPS).rsqrt().to(t)
            s["d_y"], s["d_sum"] = normal(r, c, std=1e-2), normal(r, c, std=1e-2)
            s["d_gamma"] = torch.empty(1, c, device=DEV, dtype=t)
    elif op in ("scan_fwd", "scan_bwd"):
        n, b, c = case["tokens"], case["seqs"], case["channels"]
        starts = _starts(case, seed)
        s["offsets"] = torch.tensor(starts, device=DEV).reshape(-1, 1) if case["ragged"] else None
        s["starts"] = torch.tensor(starts, device=DEV)
        s["x"], s["z"], s["h0"] = normal(n, c), normal(n, c, std=1.5, mean=2.0), normal(b, c)
        s["res"], s["last"] = torch.empty(n, c, device=DEV, dtype=t), torch.empty(b, c, device=DEV, dtype=t)
        if op == "scan_bwd":  # h: what the forward pass kept
            s["h"], _ = _scan(s["x"], s["z"], s["h0"], s["starts"])
            s["d_out"], s["d_last"] = normal(n, c, std=1e-2), normal(b, c, std=1e-2)
            s["d_z"], s["d_h0"] = torch.empty(n, c, device=DEV, dtype=t), torch.empty(b, c, device=DEV, dtype=t)
    else:
        r, k, o, gr = case["rows"], case["cols"], case["outs"], case["group"]
        ng = -(-k // gr)
        # row-major packed codes, two to a byte, the even column in the low half; one scale a group of columns
        s["codes"] = torch.randint(0, 256, (o, -(-k // 2)), generator=g, device=DEV, dtype=torch.uint8)
        s["scales"] = (torch.rand(o, ng, generator=g, device=DEV) + 0.5) * (0.15 / math.sqrt(k))
        s["x"], s["y"] = normal(r, k), torch.empty(r, o, device=DEV)
        if op == "norm_q8_q4":
            s["residual"], s["gamma"], s["h"] = normal(r, k), normal(1, k, std=0.1, mean=1.0), torch.empty(r, k, device=DEV)
            s["q"] = torch.empty(r, k, device=DEV, dtype=torch.int8)
            s["q_scale"], s["inv"] = torch.empty(r, 1, device=DEV), torch.empty(r, 1, device=DEV)
    if own:  # a user's program holds its data as the framework's matrices: views of the tensors above
        from daphne_amd.kernels import DenseMatrix

        ctx = _context()
        for k in [k for k, v in s.items() if isinstance(v, torch.Tensor) and k != "starts"]:
            m = s[k].reshape(-1, 1) if k == "ids" else s[k]
            s["m_" + k] = DenseMatrix.from_torch(ctx, m)
        s["ctx"] = ctx
    return s


_kept = {}


def _context():
    """One context for the program's life. Token numbers and offsets are checked on the device by every call; the
    verdicts are kept there until the program asks for them, as a training or serving loop does."""
    if "ctx" not in _kept:
        from daphne_amd.kernels import HIPContext

        _kept["ctx"] = HIPContext(torch.cuda.current_device())
        _kept["checks"] = _kept["ctx"].deferred_checks()
        _kept["checks"].__enter__()
    return _kept["ctx"]


# ------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------
def _affine_scan(a, b):
    """All h_t = a_t h_{t-1} + b_t (h_{-1} = 0) by doubling: after the pass with distance d, row t holds the composition
    of its last 2 d steps."""
    d = 1
    while d < a.shape[0]:
        b = torch.cat((b[:d], torch.addcmul(b[d:], a[d:], b[:-d])))
        a = torch.cat((a[:d], a[d:] * a[:-d]))
        d *= 2
    return b


def _scan(x, z, h0, starts):
    f = torch.sigmoid(z)
    b = torch.sigmoid(-z) * x
    first, end = starts[:-1], starts[1:]
    some = end > first
    b.index_add_(0, first[some], f[first[some]] * h0[some])
    h = _affine_scan(f.index_fill(0, first[some], 0.0), b)
    return h, torch.where(some[:, None], h[(end - 1).clamp_min(0)], h0)


def _scan_back(x, z, h, h0, d_out, d_last, starts):
    f, w = torch.sigmoid(z), torch.sigmoid(-z)
    first, end = starts[:-1], starts[1:]
    some = end > first
    a = torch.cat((f[1:], torch.zeros_like(f[:1]))).index_fill(0, end[some] - 1, 0.0)
    b = d_out.index_add(0, end[some] - 1, d_last[some])
    grad = _affine_scan(a.flip(0), b.flip(0)).flip(0)
    before = torch.cat((h[:1], h[:-1])).index_copy(0, first[some], h0[some])
    at = first.clamp_max(x.shape[0] - 1)
    return {"d_x": w * grad, "d_z": grad * (before - x) * f * w, "d_h0": torch.where(some[:, None], f[at] * grad[at], d_last)}


def _unpacked(codes, cols):
    lo, hi = codes & 15, codes >> 4
    return ((torch.stack((lo, hi), -1).reshape(codes.shape[0], -1)[:, :cols].to(torch.int8) ^ 8) - 8).float()


def _plain(s):
    op, c = s["op"], s["case"]
    if op == "embed_fwd":
        return s["table"][s["ids"]] * s["scale"]
    if op == "embed_bwd":  # sums over every occurrence of a frequent token: in 64 bits
        d = s["d_out"]
        acc = torch.zeros(c["vocab"], c["width"], device=DEV, dtype=torch.float64).index_add_(0, s["ids"], d.double())
        return (acc * s["scale"]).to(d.dtype)
    if op == "norm_fwd":
        h = s["x"] + s["residual"]
        inv = (h.square().mean(1, keepdim=True) + EPS).rsqrt()
        return {"y": h * inv * s["gamma"], "h": h, "inv": inv}
    if op == "norm_bwd":
        h, inv, dy = s["x"], s["inv"], s["d_y"]
        u = dy * s["gamma"]
        dx = inv * (u - h * (inv * inv * (u * h).mean(1, keepdim=True))) + s["d_sum"]
        return {"d_x": dx, "d_gamma": (dy * h * inv).sum(0, keepdim=True, dtype=torch.float64).to(h.dtype)}
    if op == "scan_fwd":
        h, last = _scan(s["x"], s["z"], s["h0"], s["starts"])
        return {"h": h, "last": last}
    if op == "scan_bwd":
        return _scan_back(s["x"], s["z"], s["h"], s["h0"], s["d_out"], s["d_last"], s["starts"])
    w = _unpacked(s["codes"], c["cols"]) * s["scales"].repeat_interleave(c["group"], 1)[:, : c["cols"]]
    if op == "q4":
        return s["x"] @ w.t()
    h = s["x"] + s["residual"]
    inv = (h.square().mean(1, keepdim=True) + EPS).rsqrt()
    u = h.double() * s["gamma"].double()  # codes next to a border: in 64 bits
    most = u.abs().amax(1, keepdim=True)
    q = torch.round(u * (127.0 / most))
    return {"y": (q.float() * (most * inv / 127.0).float()) @ w.t(), "h": h}


def _own(s):
    from daphne_amd import kernels as K

    op, c, ctx, m = s["op"], s["case"], s["ctx"], lambda k: s.get("m_" + k)
    if op == "embed_fwd":
        K.embeddingForward(m("res"), m("table"), m("ids"), s["scale"], ctx)
        return s["res"]
    if op == "embed_bwd":
        K.embeddingBackward(m("d_table"), m("d_out"), m("ids"), c["vocab"], s["scale"], ctx)
        return s["d_table"]
    if op == "norm_fwd":
        K.rmsNormForward(m("y"), m("h"), m("inv"), m("x"), m("residual"), m("gamma"), EPS, ctx)
        return {"y": s["y"], "h": s["h"], "inv": s["inv"]}
    if op == "norm_bwd":
        K.rmsNormBackward(m("y"), m("d_gamma"), m("x"), m("inv"), m("gamma"), m("d_y"), m("d_sum"), ctx)
        return {"d_x": s["y"], "d_gamma": s["d_gamma"]}
    if op == "scan_fwd":
        K.gatedRecurrenceForward(m("res"), m("last"), m("x"), m("z"), m("h0"), m("offsets"), c["seqs"], ctx)
        return {"h": s["res"], "last": s["last"]}
    if op == "scan_bwd":
        K.gatedRecurrenceBackward(m("res"), m("d_z"), m("d_h0"), m("x"), m("z"), m("h"), m("h0"), m("d_out"), m("d_last"),
                                  m("offsets"), c["seqs"], ctx)
        return {"d_x": s["res"], "d_z": s["d_z"], "d_h0": s["d_h0"]}
    if op == "q4":
        K.matVecQ4(m("y"), m("x"), None, m("codes"), m("scales"), c["group"], ctx)
        return s["y"]
    K.rmsNormForwardQ8(m("q"), m("q_scale"), m("h"), m("inv"), m("x"), m("residual"), m("gamma"), EPS, ctx)
    K.matVecQ4(m("y"), m("q"), m("q_scale"), m("codes"), m("scales"), c["group"], ctx)
    return {"y": s["y"], "h": s["h"]}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------
# work and exact values
# ------------------------------------------------------------------------------------------
def work(case):
    op, z = case["op"], 8 if case.get("type") == "f64" else 4
    if op == "embed_fwd":
        n, w = case["tokens"], case["width"]
        return {"bytes": n * 8 + (min(n, case["vocab"]) + n) * w * z, "flops": n * w}
    if op == "embed_bwd":
        n, w = case["tokens"], case["width"]
        return {"bytes": n * 8 + (case["vocab"] + n) * w * z, "flops": n * w}
    if op in ("norm_fwd", "norm_bwd"):
        e = case["rows"] * case["cols"]
        return {"bytes": 4 * e * z, "flops": (5 if op == "norm_fwd" else 9) * e}
    if op in ("scan_fwd", "scan_bwd"):
        e, b = case["tokens"] * case["channels"], case["seqs"] * case["channels"]
        return {"bytes": ((3 * e + 2 * b) if op == "scan_fwd" else (6 * e + 3 * b)) * z, "flops": (8 if op == "scan_fwd" else 14) * e}
    r, k, o = case["rows"], case["cols"], case["outs"]
    b = o * (k // 2) + o * -(-k // case["group"]) * 4 + r * o * 4
    return {"bytes": b + r * k * (4 if op == "q4" else 12), "flops": 2 * r * k * o}


def _sequential(f, b, first):
    """h_t = f_t h_{t-1} + b_t row by row; a row that begins a sequence takes the state it is given."""
    out, h = torch.empty_like(b), torch.zeros_like(b[0])
    for t in range(b.shape[0]):
        if t in first:
            h = first[t]
        h = torch.addcmul(b[t], f[t], h, out=out[t])
    return out


def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    op = case["op"]
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if op == "embed_fwd":
        return torch.index_select(d["table"], 0, s["ids"]).mul_(s["scale"])
    if op == "embed_bwd":
        order = torch.argsort(s["ids"], stable=True)
        counts = torch.bincount(s["ids"], minlength=case["vocab"])
        return torch.segment_reduce(d["d_out"][order], "sum", lengths=counts, axis=0, initial=0.0).mul_(s["scale"])
    if op in ("norm_fwd", "norm_bwd", "norm_q8_q4"):
        # the sum is a stored value of the residual stream: rounded to its type, and what follows goes by it
        stored = (d["x"] + d["residual"]).to(s["x"].dtype).double() if op != "norm_bwd" else d["x"]
        inv = 1.0 / torch.sqrt(torch.linalg.vector_norm(stored, dim=1, keepdim=True) ** 2 / stored.shape[1] + EPS)
    if op == "norm_fwd":
        return {"y": stored * d["gamma"] * inv, "h": d["x"] + d["residual"], "inv": inv}
    if op == "norm_bwd":
        inv = d["inv"]
        n = stored * inv
        u = d["d_y"] * d["gamma"]
        dot = torch.linalg.vecdot(u, n).unsqueeze(1) / n.shape[1]
        return {"d_x": (u - n * dot) * inv + d["d_sum"], "d_gamma": torch.linalg.vecdot(d["d_y"], n, dim=0).unsqueeze(0)}
    if op in ("scan_fwd", "scan_bwd"):
        if case["tokens"] > 140000:
            return None
        starts = s["starts"].tolist()
        f = 1.0 / (1.0 + torch.exp(-d["z"]))
        w = 1.0 / (1.0 + torch.exp(d["z"]))
        spans = [(i, a, e) for i, (a, e) in enumerate(zip(starts[:-1], starts[1:]))]
        if op == "scan_fwd":
            h = _sequential(f, w * d["x"], {a: d["h0"][i] for i, a, e in spans if e > a})
            last = torch.stack([h[e - 1] if e > a else d["h0"][i] for i, a, e in spans])
            return {"h": h, "last": last}
        # backwards in time, the incoming gradient of a sequence's last row being d_last, and f one row later
        grad = torch.empty_like(f)
        for i, a, e in spans:
            if e > a:
                late = torch.ones_like(f[a:e])
                late[:-1] = f[a + 1 : e]
                grad[a:e] = _sequential(late.flip(0), d["d_out"][a:e].flip(0), {0: d["d_last"][i]}).flip(0)
        prior = torch.empty_like(f)
        prior[1:] = d["h"][:-1]
        for i, a, e in spans:
            if e > a:
                prior[a] = d["h0"][i]
        d_h0 = torch.stack([f[a] * grad[a] if e > a else d["d_last"][i] for i, a, e in spans])
        return {"d_x": grad * w, "d_z": grad * (prior - d["x"]) * f * w, "d_h0": d_h0}
    k, o, gr = case["cols"], case["outs"], case["group"]
    byte = s["codes"].long()
    c = torch.empty(o, 2 * byte.shape[1], device=DEV, dtype=torch.float64)
    c[:, 0::2], c[:, 1::2] = byte % 16, byte // 16
    c = torch.where(c > 7, c - 16, c)[:, :k]
    x = d["x"]
    if op == "norm_q8_q4":
        u = stored * d["gamma"]
        most = u.abs().max(1, keepdim=True).values
        x = torch.round(u * (127.0 / most)) * (most * inv / 127.0)
    y = torch.zeros(x.shape[0], o, device=DEV, dtype=torch.float64)
    for j in range(0, k, gr):
        y += (x[:, j : j + gr] @ c[:, j : j + gr].t()) * d["scales"][:, j // gr]
    return y if op == "q4" else {"y": y, "h": d["x"] + d["residual"]}
