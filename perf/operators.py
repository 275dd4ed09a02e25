"""Cases that measure the MXFP4 expert operators: routing to experts, the
MXFP4 quantiser with its read-back, and the product of tokens with the MXFP4
matrices of the experts they picked.

`run` gives each operator in plain torch, or (with `own`) through the
package's public entry points; `exact` gives it in 64 bits, written apart.
"""
import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32            # values that share one scale
BLOCK_BYTES = 17      # one scale byte, then 16 bytes of 4-bit codes
MIN_SUM = 2.0 ** -14  # lower bound of the sum that renormalises gating weights
DEV = "cuda"

_pkg = None


def pkg():
    global _pkg
    if _pkg is None:
        _pkg = importlib.import_module("a6000-custom-kernels_b200")
    return _pkg


# ---- cases -------------------------------------------------------------------

def _route(name, n_tok, E, k, score, bias, n_group, topk_group, group_score, norm_w, scale, dtype):
    return {"name": name, "op": "route", "n_tok": n_tok, "E": E, "k": k, "score": score, "bias": bias,
            "n_group": n_group, "topk_group": topk_group, "group_score": group_score, "norm_w": norm_w,
            "scale": scale, "dtype": dtype}


def _quant(name, rows, K, planes, dtype, strided):
    return {"name": name, "op": "quant", "rows": rows, "K": K, "planes": planes, "dtype": dtype, "strided": strided}


def _product(name, n_tok, E, k, K, rows, glu, bias, per_pick, planes, dtype):
    """glu: "" for the plain product, else the GLU of the fused gate."""
    return {"name": name, "op": "product", "n_tok": n_tok, "E": E, "k": k, "K": K, "rows": rows, "glu": glu,
            "bias": bias, "per_pick": per_pick, "planes": planes, "dtype": dtype}


def listed():
    return [
        # one decode token through a router with sigmoid scores, a balance bias and groups: pure latency
        _route("route_token", 1, 256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5, "f32"),
        # a mixed batch with 16-bit logits (many equal ones) and weights from a softmax over the picks
        _route("route_batch", 77, 160, 6, "softmax_topk", False, 1, 1, "max", False, 1.0, "bf16"),
        # a long prompt through the grouped, biased router
        _route("route_prompt", 8192, 256, 8, "sigmoid", True, 8, 4, "top2", True, 2.5, "f32"),
        # the activations of one token's eight picks before the down projection, two planes
        _quant("quant_token", 8, 768, 2, "f32", False),
        # a ragged batch of rows that lie in a wider buffer, sizes off the powers of two
        _quant("quant_rows", 333, 1440, 2, "f16", True),
        # matrices brought to four bits (a checkpoint's weights, a prompt's activations)
        _quant("quant_matrix", 16384, 4096, 1, "bf16", False),
        # gate and up of one decode token with SwiGLU: the weights' bytes and latency
        _product("token_glu", 1, 64, 8, 2048, 768, "swiglu", False, False, 2, "f32"),
        # the down projection of eight decode tokens, each pick with its own row
        _product("batch_down", 8, 64, 8, 768, 2048, "", False, True, 2, "f32"),
        # a short ragged prompt, odd sizes, biases and the clamped GLU, one plane
        _product("ragged_glu", 45, 24, 4, 1440, 1000, "swiglu_oai", True, False, 1, "bf16"),
        # a prompt through gate and up
        _product("prompt_glu", 512, 64, 8, 2048, 768, "swiglu", False, False, 2, "f32"),
        # a prompt through the down projection
        _product("prompt_down", 2048, 32, 8, 768, 2048, "", False, True, 2, "f32"),
        # a batch of long prompts through gate and up, one plane
        _product("long_glu", 4096, 64, 8, 2048, 1024, "swiglu", False, False, 1, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "quant", "product", "product"])
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    if op == "route":
        n_group = rng.choice([1, 1, 2, 4, 8])
        E = n_group * rng.randint(2 if n_group > 1 else 8, 64 if n_group > 1 else 512)
        topk_group = rng.randint(1, n_group)
        k = rng.randint(1, min(16, topk_group * (E // n_group)))
        score = rng.choice(["softmax", "sigmoid", "softmax_topk"])
        c = _route("", _log_int(rng, 1, 8192), E, k, score, rng.random() < 0.6, n_group, topk_group,
                   rng.choice(["max", "top2"]), rng.random() < 0.5, rng.choice([1.0, 1.5, 2.5]), dtype)
    elif op == "quant":
        K = BLOCK * _log_int(rng, 1, 256)
        rows = _log_int(rng, 1, min(65536, 16384 * 4096 // K))
        planes = rng.choice([1, 2]) if rows * K <= 16384 * 1024 else 1
        c = _quant("", rows, K, planes, dtype, rng.random() < 0.3)
    else:
        E = _log_int(rng, 2, 128)
        k = rng.randint(1, min(8, E))
        K = BLOCK * _log_int(rng, 1, 96)
        rows = _log_int(rng, 8, 2048)
        glu = rng.choice(["", "swiglu", "geglu", "swiglu_oai"])
        per_pick = not glu and rng.random() < 0.5
        planes = rng.choice([1, 2, 2])
        top = 4096 * 64 * 2048 * 1024 * 2      # the largest listed plain product over all experts
        cost = E * K * rows * (2 if glu else 1) * (k if per_pick else 1)
        n_tok = _log_int(rng, 1, max(1, min(4096, top // (2 * cost))))
        c = _product("", n_tok, E, k, K, rows, glu, rng.random() < 0.4, per_pick, planes, dtype)
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _logits(g, n_tok, E):
    """Router logits as trained routers give them: a skew over the experts (Zipf, 1.1) and N(0, 1) per token."""
    rank = torch.randperm(E, generator=g, device=DEV).to(torch.float32)
    return -1.1 * torch.log(rank + 1.0) + torch.randn((n_tok, E), generator=g, device=DEV)


def _weights(g, E, rows, K):
    """uint8 [E][rows][17 K / 32]: N(0, 0.02) matrices in MXFP4 blocks, one expert at a time."""
    out = torch.empty((E, rows, K // BLOCK * BLOCK_BYTES), dtype=torch.uint8, device=DEV)
    for e in range(E):
        out[e] = _quantize(0.02 * torch.randn((rows, K), generator=g, device=DEV), 1)[:, 0]
    return out


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    dt = DTYPES[case["dtype"]]
    if case["op"] == "route":
        s["logits"] = _logits(g, case["n_tok"], case["E"]).to(dt)
        s["bias"] = 0.1 * torch.randn(case["E"], generator=g, device=DEV) if case["bias"] else None
    elif case["op"] == "quant":
        rows, K = case["rows"], case["K"]
        wide = K + (48 if case["strided"] else 0)
        x = torch.randn((rows, wide), generator=g, device=DEV)
        x *= torch.exp(torch.randn((rows, 1), generator=g, device=DEV))      # rows of different magnitudes
        s["x"] = x.to(dt)[:, :K]
    else:
        n, E, k, K, rows = (case[v] for v in ("n_tok", "E", "k", "K", "rows"))
        s["w"] = _weights(g, E, rows, K)
        s["gate"] = _weights(g, E, rows, K) if case["glu"] else None
        s["bias"] = 0.1 * torch.randn((E, rows), generator=g, device=DEV) if case["bias"] else None
        s["gate_bias"] = 0.1 * torch.randn((E, rows), generator=g, device=DEV) if case["bias"] and case["glu"] else None
        s["ids"] = torch.topk(_logits(g, n, E), k, dim=1)[1].to(torch.int32)
        s["x"] = torch.randn((n, k, K) if case["per_pick"] else (n, K), generator=g, device=DEV).to(dt)
        if own:   # the matrices laid out once for the kernels, as a program that loads a model keeps them
            s["w_own"] = pkg().MXFP4Weights(s["w"], K, rows)
            s["gate_own"] = pkg().MXFP4Weights(s["gate"], K, rows) if case["glu"] else None
    return s


# ---- the operators -------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["op"] == "route":
        return _route_plain(s["logits"], s["bias"], c)
    if c["op"] == "quant":
        return _dequantize(_quantize(s["x"], c["planes"]), c["K"]).to(s["x"].dtype)
    return _product_plain(s, c)


def _run_own(s, c):
    p = pkg()
    if c["op"] == "route":
        return p.route_experts(s["logits"], c["k"], score=c["score"], bias=s["bias"], n_group=c["n_group"],
                               topk_group=c["topk_group"], group_score=c["group_score"], norm_w=c["norm_w"],
                               scale=c["scale"])
    if c["op"] == "quant":
        return p.dequantize_mxfp4(p.quantize_mxfp4(s["x"], planes=c["planes"]), c["K"], dtype=s["x"].dtype)
    if not c["glu"]:
        return p.mxfp4_mul_mat_id(s["w_own"], s["x"], s["ids"], bias=s["bias"], planes=c["planes"])
    return p.mxfp4_mul_mat_id(s["w_own"], s["x"], s["ids"], gate=s["gate_own"], bias=s["bias"],
                              gate_bias=s["gate_bias"], glu_op=getattr(p.moe_cache, "GLU_" + c["glu"].upper()),
                              planes=c["planes"])


def _route_plain(logits, bias, c):
    """Scores in 32 bits; what ranks experts in 64, where a bias or a group sum can bring two of them close."""
    E, k, n_group = c["E"], c["k"], c["n_group"]
    l32 = torch.clamp(logits.float(), max=torch.finfo(torch.float32).max)
    l64 = l32.double()
    if c["score"] == "sigmoid":
        s32 = 1.0 / (1.0 + torch.exp(-l32))
        s64 = 1.0 / (1.0 + torch.exp(-l64))
    elif c["score"] == "softmax":
        e32 = torch.exp(l32 - l32.amax(1, keepdim=True))
        e64 = torch.exp(l64 - l64.amax(1, keepdim=True))
        s32 = e32 / e32.sum(1, keepdim=True)
        s64 = e64 / e64.sum(1, keepdim=True)
    else:
        s32, s64 = l32, l64
    if bias is None and n_group == 1:
        key = l64
    else:
        key = s64 if bias is None else s64 + bias.double()
    if n_group > 1:
        per = key.view(-1, n_group, E // n_group)
        if c["group_score"] == "max" or E == n_group:
            gs = per.amax(2)
        else:
            gs = torch.sort(per, dim=2, descending=True)[0][:, :, :2].sum(2)
        order = torch.sort(gs, dim=1, descending=True, stable=True)[1]
        kept = torch.zeros_like(gs, dtype=torch.bool).scatter_(1, order[:, : c["topk_group"]], True)
        key = torch.where(kept[:, :, None], per, -math.inf).reshape(-1, E)
    ids = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :k]
    w = torch.gather(s32, 1, ids)
    if c["score"] == "softmax_topk":
        w = torch.exp(w - w.amax(1, keepdim=True))
        w = w / w.sum(1, keepdim=True)
    if c["norm_w"]:
        w = w / torch.clamp(w.sum(1, keepdim=True), min=MIN_SUM)
    return ids.to(torch.int32), w * c["scale"]


def _quantize(x, planes):
    """[rows][K] -> uint8 [rows][planes][17 K / 32]; plane 1 holds what plane 0 leaves of x."""
    rows, K = x.shape
    r = x.float().reshape(rows, K // BLOCK, BLOCK)
    out = []
    for _ in range(planes):
        amax = r.abs().amax(2, keepdim=True)
        e = torch.clamp(torch.frexp(amax)[1] - 3, min=-127)                    # floor(log2 amax) - 2
        e = torch.where(amax == 0, -127, e).to(torch.int32)
        v = r.abs() * ((127 - e) << 23).view(torch.float32)                    # exact: a power of two
        code = sum((v > t).to(torch.uint8) for t in (0.25, 1.25, 2.5, 5.0))    # ties go to the even code
        code = code + sum((v >= t).to(torch.uint8) for t in (0.75, 1.75, 3.5))
        code = code | (torch.signbit(r).to(torch.uint8) << 3)
        packed = code[:, :, :16] | (code[:, :, 16:] << 4)
        out.append(torch.cat([(e + 127).to(torch.uint8), packed], 2).reshape(rows, -1))
        if planes > 1:
            r = r - _dequantize(out[-1][:, None], K).view_as(r)
    return torch.stack(out, 1)


def _dequantize(blocks, K):
    """uint8 [...][planes][17 K / 32] -> f32 [...][K], the planes added."""
    b = blocks.reshape(*blocks.shape[:-1], K // BLOCK, BLOCK_BYTES)
    e = b[..., :1].to(torch.int32)
    scale = torch.where(e == 0, 1 << 22, e << 23).view(torch.float32)
    code = torch.cat([b[..., 1:] & 15, b[..., 1:] >> 4], -1).to(torch.int32)
    m = code & 7
    mag = torch.where(m < 2, m.float() * 0.5, (2 + (m & 1)).float() * 0.25 * (1 << (m >> 1)).float())
    v = torch.where(code > 7, -mag, mag) * scale
    return v.reshape(*blocks.shape[:-1], K).sum(-2)


def _product_plain(s, c):
    """The matrices of the picks where those are fewer than the experts, else every expert for every row."""
    n, E, k, K, rows = (c[v] for v in ("n_tok", "E", "k", "K", "rows"))
    x = s["x"].reshape(-1, K)
    x = _dequantize(_quantize(x, c["planes"]), K)
    ids = s["ids"].long()

    def mul(blocks, bias):
        if n * k <= E:
            w = _dequantize(blocks[ids].unsqueeze(-2), K)                       # [n][k][rows][K]
            y = torch.matmul(w, x.view(n, -1, K, 1)).squeeze(-1)
        else:
            w = _dequantize(blocks.unsqueeze(-2), K)
            y = torch.matmul(x, w.view(E * rows, K).t()).view(-1, E, rows)
            y = y[torch.arange(x.shape[0], device=x.device)[:, None], ids.reshape(x.shape[0], -1)].view(n, k, rows)
        return y if bias is None else y + bias[ids]

    y = mul(s["w"], s["bias"])
    if not c["glu"]:
        return y
    g = mul(s["gate"], s["gate_bias"])
    if c["glu"] == "swiglu":
        return y * (g / (1.0 + torch.exp(-g)))
    if c["glu"] == "geglu":
        return y * (0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * g * (1.0 + 0.044715 * g * g))))
    g = torch.clamp(g, max=7.0)
    return (g / (1.0 + torch.exp(-1.702 * g))) * (torch.clamp(y, -7.0, 7.0) + 1.0)


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    c = case
    if c["op"] == "route":
        n, E, k = c["n_tok"], c["E"], c["k"]
        return {"bytes": n * E * SIZE[c["dtype"]] + n * k * 8 + (4 * E if c["bias"] else 0), "flops": 4 * n * E}
    if c["op"] == "quant":
        n = c["rows"] * c["K"]
        held = n * BLOCK_BYTES / BLOCK * c["planes"]
        return {"bytes": 2 * n * SIZE[c["dtype"]] + 2 * held, "flops": 4 * n * c["planes"]}
    n, E, k, K, rows = (c[v] for v in ("n_tok", "E", "k", "K", "rows"))
    mats = 2 if c["glu"] else 1
    touched = E * (1 - (1 - k / E) ** n)        # experts that some token picked, expected
    x = n * (k if c["per_pick"] else 1) * K * SIZE[c["dtype"]]
    return {"bytes": mats * touched * rows * (K * BLOCK_BYTES / BLOCK + (4 if c["bias"] else 0)) + x + 4 * n * k * (rows + 1),
            "flops": 2.0 * mats * n * k * rows * K}


# ---- 64 bits, from the definitions ---------------------------------------------

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_values(x, planes):
    """The values that the planes of x stand for: nearest of the eight magnitudes, an even code on a tie."""
    mags = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    left = x.double().reshape(-1, BLOCK)
    total = torch.zeros_like(left)
    for _ in range(planes):
        top = left.abs().amax(1)
        p = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
        p = torch.where(torch.exp2(p) > top, p - 1, p)                          # log2 may round up to a whole number
        p = torch.where(torch.exp2(p + 1) <= top, p + 1, p)
        scale = torch.exp2(torch.clamp(p - 2, min=-127.0))[:, None]
        mag = left.abs() / scale
        hi = torch.bucketize(mag.contiguous(), mags).clamp(max=7)               # the first magnitude >= mag
        lo = (hi - 1).clamp(min=0)
        below, above = mag - mags[lo], mags[hi] - mag
        take = torch.where(below < above, lo, torch.where(below > above, hi, torch.where(lo % 2 == 0, lo, hi)))
        got = torch.sign(left) * mags[take] * scale
        total = total + got
        left = left - got
    return total.view(x.shape)


def _exact_matrix(blocks, K):
    """One matrix of blocks in 64 bits."""
    mags = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=blocks.device)
    b = blocks.reshape(blocks.shape[0], K // BLOCK, BLOCK_BYTES)
    both = torch.stack([b[:, :, 1:] % 16, b[:, :, 1:] // 16], 2).long()         # values 0..15, then 16..31
    return (mags[both] * torch.exp2(b[:, :, :1].double() - 127)[..., None]).reshape(blocks.shape[0], K)


def _exact_route(s, c):
    l = s["logits"].double()
    prob = torch.softmax(l, 1) if c["score"] == "softmax" else torch.sigmoid(l) if c["score"] == "sigmoid" else l
    rank = l if s["bias"] is None and c["n_group"] == 1 else prob if s["bias"] is None else prob + s["bias"].double()
    rows, w = rank.cpu(), torch.zeros((c["n_tok"], c["k"]), dtype=torch.float64)
    prob = prob.cpu()
    size = c["E"] // c["n_group"]
    for t in range(c["n_tok"]):
        r = rows[t].tolist()
        groups = [r[i * size: (i + 1) * size] for i in range(c["n_group"])]
        worth = [max(v) if c["group_score"] == "max" or size == 1 else sum(sorted(v)[-2:]) for v in groups]
        best = sorted(range(len(worth)), key=lambda i: (-worth[i], i))[: c["topk_group"]]
        pool = [e for i in best for e in range(i * size, (i + 1) * size)]
        picks = sorted(pool, key=lambda e: (-r[e], e))[: c["k"]]
        w[t] = prob[t][picks]
    if c["score"] == "softmax_topk":
        w = torch.softmax(w, 1)
    if c["norm_w"]:
        w = w / torch.clamp(w.sum(1, keepdim=True), min=MIN_SUM)
    return [None, (w * c["scale"]).to(DEV)]


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "route":
        return _exact_route(s, c)
    if c["op"] == "quant":
        return _exact_values(s["x"].contiguous(), c["planes"])
    n, E, k, K, rows = (c[v] for v in ("n_tok", "E", "k", "K", "rows"))
    x = _exact_values(s["x"].contiguous(), c["planes"]).reshape(-1, K)
    flat = s["ids"].reshape(-1).long()
    out = []
    for blocks, bias in ((s["w"], s["bias"]), (s["gate"], s["gate_bias"])):
        if blocks is None:
            continue
        y = torch.empty((n * k, rows), dtype=torch.float64, device=DEV)
        for e in range(E):
            at = torch.nonzero(flat == e).reshape(-1)
            if at.numel():
                y[at] = x[at if c["per_pick"] else at // k] @ _exact_matrix(blocks[e], K).t()
        out.append(y if bias is None else y + bias.double()[flat])
    y = out[0]
    if c["glu"] == "swiglu":
        y = out[0] * out[1] * torch.sigmoid(out[1])
    elif c["glu"] == "geglu":
        y = out[0] * torch.nn.functional.gelu(out[1], approximate="tanh")
    elif c["glu"] == "swiglu_oai":
        g = torch.clamp(out[1], max=7.0)
        y = g * torch.sigmoid(1.702 * g) * (torch.clamp(out[0], -7.0, 7.0) + 1.0)
    return y.view(n, k, rows)
