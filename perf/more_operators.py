"""Cases that measure tokens sorted by expert and back (with its gradient), and
the products with 4-bit matrices whose scales cover groups of values.

`run` gives each operator in plain torch, or (with `own`) through the
package's public entry points; `exact` gives it in 64 bits, written apart.
"""
import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"

_pkg = None


def pkg():
    global _pkg
    if _pkg is None:
        _pkg = importlib.import_module("a6000-custom-kernels_b200")
    return _pkg


# ---- cases -------------------------------------------------------------------

def _trip(name, train, n_tok, E, k, H, drop, shared, dtype):
    """Tokens to their experts' rows and back; with `train` the gradients too. `drop`: share of picks without an expert."""
    return {"name": name, "op": "train" if train else "trip", "n_tok": n_tok, "E": E, "k": k, "H": H, "drop": drop,
            "shared": shared, "dtype": dtype}


def _w4(name, n_tok, E, k, K, rows, group, zeros, glu, bias, per_pick, dtype, scale_dtype):
    """E = 0: one matrix for all tokens. glu: "" for the plain product, else the GLU of the fused gate."""
    return {"name": name, "op": "w4", "n_tok": n_tok, "E": E, "k": k, "K": K, "rows": rows, "group": group, "zeros": zeros,
            "glu": glu, "bias": bias, "per_pick": per_pick, "dtype": dtype, "scale_dtype": scale_dtype}


def listed():
    return [
        # one decode token to its eight experts and back, the shared expert added: pure latency
        _trip("trip_token", False, 1, 64, 8, 2048, 0.0, True, "f32"),
        # a ragged decode batch, sizes off the powers of two, a tenth of the picks held elsewhere
        _trip("trip_batch", False, 77, 160, 6, 1442, 0.1, False, "f16"),
        # a long prompt
        _trip("trip_prompt", False, 8192, 64, 8, 2048, 0.0, False, "bf16"),
        # a small training batch in 32 bits, odd sizes, some picks over an expert's capacity
        _trip("train_batch", True, 333, 24, 4, 1000, 0.05, False, "f32"),
        # a training step's tokens over many experts
        _trip("train_long", True, 16384, 256, 8, 2048, 0.0, False, "bf16"),
        # one token through one small matrix (a shared expert's projection): latency
        _w4("vec_token", 1, 0, 1, 2048, 768, 128, False, "", False, False, "f32", "f16"),
        # one token through the largest matrix (an output head), with zeros: the weights' bytes
        _w4("vec_head", 1, 0, 1, 4096, 32768, 64, True, "", False, False, "bf16", "bf16"),
        # a few tokens, a K that ends inside a group, odd sizes, a bias
        _w4("vec_ragged", 5, 0, 1, 1446, 1000, 128, True, "", True, False, "f32", "f16"),
        # a decode batch through one matrix with small groups
        _w4("vec_batch", 24, 0, 1, 4096, 4096, 32, True, "", False, False, "f16", "f16"),
        # gate and up of one decode token's experts with SwiGLU
        _w4("experts_token", 1, 64, 8, 2048, 768, 128, False, "swiglu", False, False, "f32", "f16"),
        # the down projection of eight decode tokens, each pick with its own row
        _w4("experts_down", 8, 64, 8, 768, 2048, 32, False, "", False, True, "f32", "f16"),
        # a large decode batch through gate and up, biases and the clamped GLU
        _w4("experts_batch", 64, 64, 8, 2048, 1024, 128, True, "swiglu_oai", True, False, "bf16", "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "f16"])
    if rng.random() < 0.45:
        train = rng.random() < 0.5
        E = _log_int(rng, 2, 512)
        k = rng.randint(1, min(12, E))
        H = _log_int(rng, 16, 8192)
        most = 16384 * 8 * 2048 * 2 // (k * H * SIZE[dtype])       # the rows of the largest listed case
        c = _trip("", train, _log_int(rng, 1, max(1, min(32768, most))), E, k, H, rng.choice([0.0, 0.0, 0.05, 0.3]),
                  not train and rng.random() < 0.4, dtype)
    else:
        E = rng.choice([0, _log_int(rng, 2, 128)])
        k = rng.randint(1, min(8, E)) if E else 1
        K = 2 * _log_int(rng, 16, 4096)
        glu = rng.choice(["", "", "swiglu", "geglu", "swiglu_oai"]) if E else ""
        most = 64 * 2048 * 1024 * 2 // (max(1, E) * K * (2 if glu else 1))   # the values of the largest listed case
        c = _w4("", _log_int(rng, 1, 64), E, k, K, _log_int(rng, 8, max(8, min(32768 if not E else 4096, most))),
                rng.choice([32, 64, 128, 128, 256]), rng.random() < 0.5, glu, rng.random() < 0.3,
                bool(E) and not glu and rng.random() < 0.5, dtype, rng.choice(["f16", "bf16"]))
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _ids(g, n_tok, E, k):
    """The picks of router logits as trained routers give them: a skew over the experts (Zipf, 1.1) and N(0, 1) per token."""
    rank = torch.randperm(E, generator=g, device=DEV).to(torch.float32)
    logits = -1.1 * torch.log(rank + 1.0) + _randn(g, n_tok, E)
    top, ids = torch.topk(logits, k, dim=1)
    return ids.to(torch.int32), torch.softmax(top, 1)


def _matrices(g, E, rows, K, group, zeros, dtype):
    """N(0, 0.02) matrices in 4 bits: codes uint8 [E][rows][K / 2] (value 2 i in the low nibble of byte i), scales and
    zeros [E][rows][groups], one expert at a time."""
    n = -(-K // group)
    codes = torch.empty((E, rows, K // 2), dtype=torch.uint8, device=DEV)
    scales = torch.empty((E, rows, n), dtype=dtype, device=DEV)
    zs = torch.empty((E, rows, n), dtype=torch.uint8, device=DEV) if zeros else None
    for e in range(E):
        w = torch.nn.functional.pad(0.02 * _randn(g, rows, K), (0, n * group - K)).view(rows, n, group)
        if zeros:
            lo, hi = w.amin(2), w.amax(2)
            scales[e] = ((hi - lo) / 15.0).to(dtype)
            s = scales[e].float()
            zs[e] = torch.clamp(torch.round(-lo / s), 0, 15).to(torch.uint8)
            z = zs[e].float()
        else:
            scales[e] = (w.abs().amax(2) / 7.5).to(dtype)
            s, z = scales[e].float(), 8.0
        q = torch.round(w / s[..., None]) + (z[..., None] if zeros else z)
        q = torch.clamp(q, 0, 15).to(torch.uint8).view(rows, n * group)[:, :K]
        codes[e] = q[:, 0::2] | (q[:, 1::2] << 4)
    return codes, scales, zs


def prepare(case, seed):
    g = _gen(seed)
    c = case
    s = {"case": c}
    dt = DTYPES[c["dtype"]]
    n, E, k = c["n_tok"], c["E"], c["k"]
    if c["op"] == "w4":
        K, rows = c["K"], c["rows"]
        first = max(1, E)
        mats = {"w": _matrices(g, first, rows, K, c["group"], c["zeros"], DTYPES[c["scale_dtype"]])}
        if c["glu"]:
            mats["gate"] = _matrices(g, first, rows, K, c["group"], c["zeros"], DTYPES[c["scale_dtype"]])
        s["bias"] = 0.1 * _randn(g, first, rows) if c["bias"] else None
        s["gate_bias"] = 0.1 * _randn(g, first, rows) if c["bias"] and c["glu"] else None
        s["x"] = _randn(g, *((n, k, K) if c["per_pick"] else (n, K))).to(dt)
        s["ids"] = _ids(g, n, E, k)[0] if E else torch.zeros((n, 1), dtype=torch.int32, device=DEV)
        s["mats"] = mats
        if own:   # laid out once for the kernels, as a program that loads a model keeps them
            s["own"] = {r: pkg().W4Weights(m[0], m[1], K, c["group"], zeros=m[2]) for r, m in mats.items()}
        return s
    s["ids"], w = _ids(g, n, E, k)
    if c["drop"]:
        s["ids"][torch.rand((n, k), generator=g, device=DEV) < c["drop"]] = -1
    s["weights"] = w
    s["x"] = _randn(g, n, c["H"]).to(dt)
    s["y"] = _randn(g, n * k, c["H"]).to(dt)       # the experts' outputs, a row for each sorted pick
    s["shared"] = _randn(g, n, c["H"]).to(dt) if c["shared"] else None
    if c["op"] == "train":
        s["d_rows"] = _randn(g, n * k, c["H"]).to(dt)
        s["d_out"] = _randn(g, n, c["H"]).to(dt)
        for v in ("x", "y", "weights"):
            s[v].requires_grad_()
    return s


# ---- the operators -------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["op"] == "w4":
        return _product_plain(s, c)
    return _trip_plain(s, c)


def _run_own(s, c):
    p = pkg()
    if c["op"] == "w4":
        w = s["own"]
        if not c["E"]:
            return p.w4_mul_mat(w["w"], s["x"], bias=s["bias"])
        if not c["glu"]:
            return p.w4_mul_mat_id(w["w"], s["x"], s["ids"], bias=s["bias"])
        return p.w4_mul_mat_id(w["w"], s["x"], s["ids"], gate=w["gate"], bias=s["bias"], gate_bias=s["gate_bias"],
                               glu_op=getattr(p.moe_cache, "GLU_" + c["glu"].upper()))
    rows, order = p.dispatch_sorted(s["x"], s["ids"], c["E"])
    out = p.combine_sorted(s["y"], order, s["weights"], shared=s["shared"])
    where = {"rows": order.rows, "positions": order.positions, "offsets": order.offsets}
    if c["op"] == "trip":
        return {"x": rows, "out": out, **where}
    d_x, d_y, d_w = torch.autograd.grad([rows, out], [s["x"], s["y"], s["weights"]], [s["d_rows"], s["d_out"]])
    return {"x": rows.detach(), "out": out.detach(), "d_x": d_x, "d_y": d_y, "d_w": d_w, **where}


def _trip_plain(s, c):
    n, E, k, H = c["n_tok"], c["E"], c["k"], c["H"]
    dt, ids = s["x"].dtype, s["ids"].reshape(-1)
    x, y, w = s["x"].detach(), s["y"].detach(), s["weights"].detach()
    held = ids >= 0
    order = torch.sort(torch.where(held, ids, E), stable=True)[1]
    counts = torch.zeros(E + 1, dtype=torch.int64, device=ids.device)
    counts.index_add_(0, torch.where(held, ids, E).long(), torch.ones_like(order))
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts[:E], 0)])
    live = held[order]                                              # the sorted rows that hold a pick
    positions = torch.empty_like(order).scatter_(0, order, torch.arange(n * k, device=ids.device))
    rows = torch.where(live[:, None], x[order // k], torch.zeros((), dtype=dt, device=x.device))
    y_of = torch.where(held[:, None], y[positions].float(), 0.0).view(n, k, H)
    out = (y_of * w[:, :, None]).sum(1)
    if s["shared"] is not None:
        out = out + s["shared"].float()
    got = {"x": rows, "out": out.to(dt), "rows": torch.where(live, order, -1).to(torch.int32),
           "positions": torch.where(held, positions, -1).to(torch.int32).view(n, k), "offsets": offsets.to(torch.int32)}
    if c["op"] == "train":
        d_out = s["d_out"].float()
        got["d_w"] = (y_of * d_out[:, None, :]).sum(2)
        del y_of
        d_y = d_out[order // k] * w.reshape(-1)[order][:, None]
        got["d_y"] = torch.where(live[:, None], d_y, 0.0).to(dt)
        del d_y
        got["d_x"] = torch.where(held[:, None], s["d_rows"][positions].float(), 0.0).view(n, k, H).sum(1).to(dt)
    return got


def _values(mat, K, group):
    codes, scales, zeros = mat
    q = torch.stack([codes & 15, codes >> 4], -1).view(*codes.shape[:-1], K).float()
    z = 8.0 if zeros is None else torch.repeat_interleave(zeros.float(), group, -1)[..., :K]
    return (q - z) * torch.repeat_interleave(scales.float(), group, -1)[..., :K]


def _product_plain(s, c):
    """The matrices of the picks where those are fewer than the experts, else every expert for every row."""
    n, E, k, K, rows = c["n_tok"], c["E"], c["k"], c["K"], c["rows"]
    x = s["x"].float().reshape(-1, K)
    ids = s["ids"].long()

    def mul(mat, bias):
        if not E:
            y = torch.matmul(x, _values(mat, K, c["group"])[0].t())
            return y if bias is None else y + bias
        if n * k <= E:
            w = _values([None if m is None else m[ids] for m in mat], K, c["group"])       # [n][k][rows][K]
            y = torch.matmul(w, x.view(n, -1, K, 1)).squeeze(-1)
        else:
            w = _values(mat, K, c["group"])
            y = torch.matmul(x, w.view(E * rows, K).t()).view(-1, E, rows)
            y = y[torch.arange(x.shape[0], device=x.device)[:, None], ids.reshape(x.shape[0], -1)].view(n, k, rows)
        return y if bias is None else y + bias[ids]

    y = mul(s["mats"]["w"], s["bias"])
    if not c["glu"]:
        return y
    g = mul(s["mats"]["gate"], s["gate_bias"])
    if c["glu"] == "swiglu":
        return y * (g / (1.0 + torch.exp(-g)))
    if c["glu"] == "geglu":
        return y * (0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * g * (1.0 + 0.044715 * g * g))))
    g = torch.clamp(g, max=7.0)
    return (g / (1.0 + torch.exp(-1.702 * g))) * (torch.clamp(y, -7.0, 7.0) + 1.0)


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    c = case
    n, E, k = c["n_tok"], c["E"], c["k"]
    if c["op"] != "w4":
        row = c["H"] * SIZE[c["dtype"]]
        where = n * k * 4 * 3 + 4 * (E + 1)                  # ids read, rows and positions written, offsets
        trips = (2 + 2 * k) * n * row + 4 * n * k + (n * row if c["shared"] else 0)
        if c["op"] == "train":
            trips += (2 + 3 * k) * n * row + 8 * n * k
        return {"bytes": where + trips, "flops": n * k * c["H"] * (2 if c["op"] == "trip" else 6)}
    K, rows = c["K"], c["rows"]
    mats = 2 if c["glu"] else 1
    touched = E * (1 - (1 - k / E) ** n) if E else 1         # matrices that some token picked, expected
    per = rows * (K / 2 + -(-K // c["group"]) * (2.5 if c["zeros"] else 2) + (4 if c["bias"] else 0))
    x = n * (k if c["per_pick"] else 1) * K * SIZE[c["dtype"]]
    return {"bytes": mats * touched * per + x + 4 * n * k * (rows + (1 if E else 0)), "flops": 2.0 * mats * n * k * rows * K}


# ---- 64 bits, from the definitions ---------------------------------------------

def _exact_trip(s, c):
    n, E, k, H = c["n_tok"], c["E"], c["k"], c["H"]
    flat = s["ids"].reshape(-1)
    x, y, w = s["x"].detach(), s["y"].detach(), s["weights"].detach().reshape(-1).double()
    got = {"x": torch.zeros((n * k, H), dtype=torch.float64, device=DEV), "rows": None, "positions": None, "offsets": None}
    got["out"] = torch.zeros((n, H), dtype=torch.float64, device=DEV) if s["shared"] is None else s["shared"].double().clone()
    if c["op"] == "train":
        got["d_x"] = torch.zeros((n, H), dtype=torch.float64, device=DEV)
        got["d_y"] = torch.zeros((n * k, H), dtype=torch.float64, device=DEV)
        got["d_w"] = torch.zeros(n * k, dtype=torch.float64, device=DEV)
    at = 0
    for e in range(E):
        picks = torch.nonzero(flat == e).reshape(-1)               # in order of the tokens
        t, span = picks // k, slice(at, at + picks.numel())
        at += picks.numel()
        got["x"][span] = x[t].double()
        got["out"].index_add_(0, t, w[picks][:, None] * y[span].double())
        if c["op"] == "train":
            d = s["d_out"][t].double()
            got["d_y"][span] = w[picks][:, None] * d
            got["d_w"][picks] = (d * y[span].double()).sum(1)
            got["d_x"].index_add_(0, t, s["d_rows"][span].double())
    if c["op"] == "train":
        got["d_w"] = got["d_w"].view(n, k)
    return got


def _exact_matrix(mat, e, K, group):
    codes, scales, zeros = (None if m is None else m[e] for m in mat)
    w = torch.empty((codes.shape[0], K), dtype=torch.float64, device=codes.device)
    w[:, 0::2] = (codes % 16).double()
    w[:, 1::2] = (codes // 16).double()
    for i in range(scales.shape[1]):
        part = w[:, i * group: (i + 1) * group]
        part -= 8.0 if zeros is None else zeros[:, i: i + 1].double()
        part *= scales[:, i: i + 1].double()
    return w


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] != "w4":
        return _exact_trip(s, c)
    n, E, k, K, rows = c["n_tok"], c["E"], c["k"], c["K"], c["rows"]
    x = s["x"].double().reshape(-1, K)
    flat = s["ids"].reshape(-1).long()
    out = []
    for role, bias in (("w", s["bias"]), ("gate", s["gate_bias"])):
        if role not in s["mats"]:
            continue
        y = torch.empty((n * k, rows), dtype=torch.float64, device=DEV)
        for e in range(max(1, E)):
            at = torch.nonzero(flat == e).reshape(-1)
            if at.numel():
                y[at] = x[at if c["per_pick"] else at // k] @ _exact_matrix(s["mats"][role], e, K, c["group"]).t()
        out.append(y if bias is None else y + bias.double()[flat])
    y = out[0]
    if c["glu"] == "swiglu":
        y = out[0] * out[1] * torch.sigmoid(out[1])
    elif c["glu"] == "geglu":
        y = out[0] * torch.nn.functional.gelu(out[1], approximate="tanh")
    elif c["glu"] == "swiglu_oai":
        g = torch.clamp(out[1], max=7.0)
        y = g * torch.sigmoid(1.702 * g) * (torch.clamp(out[0], -7.0, 7.0) + 1.0)
    return y.view(n, k, rows) if E else y
