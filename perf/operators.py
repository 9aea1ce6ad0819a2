"""Operators of models served and tuned in 8-bit integers, next to their plain forms.

Families (`case["op"]`):
  linear    a projection in 8-bit integers: the activations are quantized per token, the product
            with the int8 weight is scaled by token and by output channel
  qkv       the same with the activations quantized once for three projections
  experts   the feed-forward experts of an MoE layer in 8-bit integers: tokens sorted by expert and
            quantized, gate and up, SwiGLU, quantized again, down, and the weighted way back
  moe_grad  the backward pass of sorting tokens by expert and of the weighted way back: gradients of
            the experts' outputs, of the routing weights, of the router's logits and of the tokens
`own` false: the plain form, elementary torch operations in 32 bits.  `own` true: the calls of
`layerstormgemmkernels_b200.ops`.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------
def listed():
    return [
        # smallest call: one 4096 x 4096 projection for one token of a single sequence
        {"name": "linear_m1", "op": "linear", "M": 1, "N": 4096, "K": 4096, "out": "bf16"},
        # batched decoding of eight sequences, the up projection of a decoder layer
        {"name": "linear_m8", "op": "linear", "M": 8, "N": 14336, "K": 4096, "out": "bf16"},
        # a batch of sequences, or of speculated tokens, through the long K of a down projection
        {"name": "linear_m77_fp16", "op": "linear", "M": 77, "N": 4096, "K": 14336, "out": "fp16"},
        # a full prompt chunk
        {"name": "linear_m4096", "op": "linear", "M": 4096, "N": 14336, "K": 4096, "out": "bf16"},
        # q, k and v of three sequences, unrounded results
        {"name": "qkv_m3_fp32", "op": "qkv", "M": 3, "N": 4096, "N_kv": 1024, "K": 4096, "out": "fp32"},
        # q, k and v of a ragged prompt chunk, a vocabulary-like odd number of columns for q
        {"name": "qkv_m1001", "op": "qkv", "M": 1001, "N": 4099, "N_kv": 1024, "K": 4096, "out": "bf16"},
        # experts of one token (128 experts, top-8), of a decode batch, and of a prompt chunk with few wide experts
        {"name": "experts_t1", "op": "experts", "T": 1, "E": 128, "top_k": 8, "H": 2048, "I": 768},
        {"name": "experts_t64", "op": "experts", "T": 64, "E": 128, "top_k": 8, "H": 2048, "I": 768},
        {"name": "experts_t4096", "op": "experts", "T": 4096, "E": 8, "top_k": 2, "H": 4096, "I": 14336},
        # tuning the router: a short batch with an odd row length, one in 32 bits, a full training batch
        {"name": "moe_grad_t100", "op": "moe_grad", "T": 100, "E": 64, "top_k": 6, "H": 1001, "type": "bf16"},
        {"name": "moe_grad_t1024_fp32", "op": "moe_grad", "T": 1024, "E": 8, "top_k": 2, "H": 4096, "type": "fp32"},
        {"name": "moe_grad_t16384", "op": "moe_grad", "T": 16384, "E": 128, "top_k": 8, "H": 2048, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    """Spread over the logarithm of lo..hi, odd numbers among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "qkv", "experts", "experts", "moe_grad", "moe_grad"])
    if op == "linear":
        return {"op": op, "M": _log(rng, 1, 4096), "N": _log(rng, 500, 14336), "K": 16 * _log(rng, 32, 896),
                "out": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if op == "qkv":
        return {"op": op, "M": _log(rng, 1, 2048), "N": _log(rng, 1024, 8192), "N_kv": _log(rng, 256, 2048),
                "K": 16 * _log(rng, 64, 512), "out": rng.choice(["bf16", "fp16", "fp32"])}
    if op == "experts":
        # decode steps and prompts, few wide or many narrow experts
        E, k, H, I = rng.choice([(128, 8, 2048, 768), (64, 6, 2048, 1024), (32, 4, 2048, 1536), (8, 2, 4096, 14336)])
        return {"op": op, "T": _log(rng, 1, 4000), "E": E, "top_k": k, "H": H, "I": I}
    E, k = rng.choice([(128, 8), (64, 6), (32, 4), (8, 2)])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    H = rng.choice([1001, 1536, 2048, 2880, 4096])
    most = 16000 * 8 * 2048 // (k * H * (2 if kind == "fp32" else 1))
    return {"op": op, "T": _log(rng, 16, most), "E": E, "top_k": k, "H": H, "type": kind}


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------
def _randn(gen, *shape):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, 1.0, generator=gen)


def _activations(gen, rows, K):
    """bf16 [rows, K]: N(0, 1) with a few channels five times as wide, as hidden states have them."""
    wide = torch.ones(K, device="cuda")
    wide[torch.randperm(K, device="cuda", generator=gen)[: max(1, K // 256)]] = 5.0
    return (_randn(gen, rows, K) * wide).to(torch.bfloat16)


def _weight(gen, rows, K):
    """(int8 [rows, K], fp32 [rows]): the codes of N(0, 0.02) rows whose largest value is about 3.5 of that."""
    codes = torch.empty((rows, K), dtype=torch.int8, device="cuda")
    piece = max(1, (1 << 26) // K)
    for r in range(0, rows, piece):
        n = min(piece, rows - r)
        codes[r:r + n] = (_randn(gen, n, K) * 36.0).round_().clamp_(-127, 127).to(torch.int8)
    scales = torch.empty(rows, dtype=torch.float32, device="cuda").uniform_(0.8, 1.25, generator=gen) * (0.02 / 36.0)
    return codes, scales


def _routing(gen, T, E, k):
    """Top-k of random logits: (idx int32 [T, k], weights fp32 [T, k], offsets int32 [E + 1], perm, inv int32 [T k], counts)."""
    w, idx = torch.softmax(_randn(gen, T, E), -1).topk(k)
    flat = idx.flatten()
    perm = torch.sort(flat, stable=True).indices
    inv = torch.empty_like(perm)
    inv[perm] = torch.arange(T * k, device="cuda")
    counts = torch.bincount(flat, minlength=E)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    weights = (w / w.sum(-1, keepdim=True)).contiguous()
    return idx.int().contiguous(), weights, offsets, perm.int(), inv.int(), counts


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "linear":
        s["x"] = _activations(gen, case["M"], case["K"])
        s["w"], s["ws"] = _weight(gen, case["N"], case["K"])
    elif case["op"] == "qkv":
        s["x"] = _activations(gen, case["M"], case["K"])
        s["proj"] = [_weight(gen, n, case["K"]) for n in (case["N"], case["N_kv"], case["N_kv"])]
    elif case["op"] == "experts":
        T, E, k, H, I = (case[n] for n in ("T", "E", "top_k", "H", "I"))
        s["x"] = _activations(gen, T, H)
        s["idx"], s["weights"], s["offsets"], s["perm"], s["inv"], counts = _routing(gen, T, E, k)
        s["cap"] = int(counts.max())
        w, ws = _weight(gen, E * 2 * I, H)
        s["gate_up"], s["gate_up_scales"] = w.view(E, 2 * I, H), ws.view(E, 2 * I)
        w, ws = _weight(gen, E * H, I)
        s["down"], s["down_scales"] = w.view(E, H, I), ws.view(E, H)
    else:
        T, E, k, H, dt = case["T"], case["E"], case["top_k"], case["H"], DTYPES[case["type"]]
        s["idx"], s["weights"], _, _, s["inv"], _ = _routing(gen, T, E, k)
        s["y"] = _randn(gen, T * k, H).to(dt)
        s["grad_out"] = (_randn(gen, T, H) * 0.01).to(dt)
        s["grad_rows"] = (_randn(gen, T * k, H) * 0.01).to(dt)
    return s


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------
def _codes(x):
    """fp32 [..., K] -> (whole numbers -127..127 as fp32, scale fp32 [..., 1])."""
    top = x.abs().amax(-1, keepdim=True)
    return torch.round(x * 127.0 / top), top / 127.0


def _product(q, s, w, ws):
    return (q @ w.float().t()) * s * ws


def _plain_experts(s):
    T, E, k, H, I = (s[n] for n in ("T", "E", "top_k", "H", "I"))
    q, sc = _codes(s["x"].float())
    pair = s["perm"].long()
    token, expert = pair // k, s["idx"].flatten().long()[pair]
    q, sc = q[token], sc[token]
    if T * k <= E:      # few rows: the matrices of each row's expert
        at, size = None, None
        gate_up, down = s["gate_up"][expert].float(), s["down"][expert].float()
        gu = torch.bmm(gate_up, q.unsqueeze(-1)).squeeze(-1)
    else:               # every expert's rows padded to the longest expert's
        at = expert * s["cap"] + (torch.arange(T * k, device="cuda") - s["offsets"].long()[expert])
        size = E * s["cap"]
        padded = torch.zeros(size, H, device="cuda").index_copy_(0, at, q).view(E, s["cap"], H)
        gu = torch.bmm(padded, s["gate_up"].float().transpose(1, 2)).view(size, 2 * I)[at]
    gu = gu * sc * s["gate_up_scales"][expert]
    g, u = gu[:, :I], gu[:, I:]
    q, sc = _codes(g / (1.0 + torch.exp(-g)) * u)
    if at is None:
        rows = torch.bmm(down, q.unsqueeze(-1)).squeeze(-1)
    else:
        padded = torch.zeros(size, I, device="cuda").index_copy_(0, at, q).view(E, s["cap"], I)
        rows = torch.bmm(padded, s["down"].float().transpose(1, 2)).view(size, H)[at]
    rows = rows * sc * s["down_scales"][expert]
    out = (rows[s["inv"].long()].view(T, k, H) * s["weights"].unsqueeze(-1)).sum(1)
    return {"rows": rows.to(torch.bfloat16), "out": out.to(torch.bfloat16)}


def _plain_moe_grad(s):
    T, E, k, H = s["T"], s["E"], s["top_k"], s["H"]
    inv, dt, w = s["inv"].long(), s["y"].dtype, s["weights"]
    dout = s["grad_out"].float().unsqueeze(1)
    grad_y = torch.empty_like(s["y"])
    grad_y[inv] = (dout * w.unsqueeze(-1)).view(T * k, H).to(dt)
    grad_w = (s["y"][inv].float().view(T, k, H) * dout).sum(-1)
    grad_sel = w * (grad_w - (w * grad_w).sum(-1, keepdim=True))
    grad_logits = torch.zeros(T, E, device="cuda").scatter_(1, s["idx"].long(), grad_sel)
    grad_hidden = s["grad_rows"][inv].float().view(T, k, H).sum(1).to(dt)
    return {"grad_y": grad_y, "grad_weights": grad_w, "grad_logits": grad_logits, "grad_hidden": grad_hidden}


def run(s):
    if own:
        return _own(s)
    if s["op"] == "linear":
        return _product(*_codes(s["x"].float()), s["w"], s["ws"]).to(DTYPES[s["out"]])
    if s["op"] == "qkv":
        q, sc = _codes(s["x"].float())
        return [_product(q, sc, w, ws).to(DTYPES[s["out"]]) for w, ws in s["proj"]]
    return _plain_experts(s) if s["op"] == "experts" else _plain_moe_grad(s)


def _own(s):
    from layerstormgemmkernels_b200 import ops

    if s["op"] == "linear":
        return ops.int8_gemm_from_bf16(s["x"], s["w"], s["ws"], s["out"])
    if s["op"] == "qkv":
        codes, scales = ops.dynamic_int8_quant(s["x"])
        return [ops.int8_gemm(codes, w, scales, ws, s["M"], w.size(0), s["K"], s["out"]) for w, ws in s["proj"]]
    if s["op"] == "experts":
        # the rows stay in fp32 until they are combined, as in the plain form: rounded to bf16 in front of
        # the weighted sum they leave the output sqrt(2) times as far off
        rows = ops.int8_moe_ffn(s["x"], s["offsets"], s["inv"], s["top_k"], s["gate_up"], s["gate_up_scales"],
                                s["down"], s["down_scales"], "fp32")
        return {"rows": rows.to(torch.bfloat16), "out": ops.moe_unpermute(rows, s["inv"], s["weights"], "bf16")}
    grad_y, grad_w = ops.moe_unpermute_backward(s["grad_out"], s["y"], s["inv"], s["weights"])
    return {"grad_y": grad_y, "grad_weights": grad_w,
            "grad_logits": ops.moe_route_backward(s["idx"], s["weights"], grad_w, s["E"]),
            "grad_hidden": ops.moe_permute_backward(s["grad_rows"], s["inv"], s["top_k"])}


# ---------------------------------------------------------------------------------------
# Work, and the values in 64 bits
# ---------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op in ("linear", "qkv"):
        M, K, out = case["M"], case["K"], DTYPES[case["out"]].itemsize
        N = case["N"] + 2 * case.get("N_kv", 0)
        return {"bytes": N * (K + 4) + M * K * 2 + M * N * out, "flops": 2 * M * N * K}
    T, E, k, H = (case[n] for n in ("T", "E", "top_k", "H"))
    if op == "experts":
        I = case["I"]
        hit = E * (1 - (1 - k / E) ** T)      # experts that some token is routed to
        ends = T * H * 2 + T * k * (H * 2 + 4 + 8) + T * H * 2
        return {"bytes": hit * (3 * H * I + 4 * (2 * I + H)) + ends, "flops": 6 * T * k * H * I}
    size = DTYPES[case["type"]].itemsize
    # read: grad_out, y, grad_rows, inv, weights, idx; written: grad_y, grad_hidden, grad_weights, grad_logits
    return {"bytes": (2 * T * H + 3 * T * k * H) * size + T * k * 16 + T * E * 4, "flops": T * k * (4 * H + 5)}


def _exact_codes(x):
    top = x.abs().max(dim=-1, keepdim=True).values
    return (x / (top / 127.0)).mul(2.0 ** 20).round().div(2.0 ** 20).round(), top / 127.0


def exact(case, seed):
    """The definitions in 64 bits.  (A quotient of bf16 values that is not half-way between two codes is
    further than 2^-20 from being so; rounding it there first keeps half-way ones where they are.)"""
    s = prepare(case, seed)
    if case["op"] in ("linear", "qkv"):
        q, sc = _exact_codes(s["x"].double())
        outs = [(sc * torch.mm(q, w.double().t()) * ws.double()[None]) for w, ws in s.get("proj", [(s.get("w"), s.get("ws"))])]
        return outs if case["op"] == "qkv" else outs[0]
    T, k, H = case["T"], case["top_k"], case["H"]
    if case["op"] == "experts":
        I, offsets = case["I"], s["offsets"].tolist()
        q, sc = _exact_codes(s["x"].double())
        rows = torch.empty(T * k, H, dtype=torch.float64, device="cuda")
        for e in range(case["E"]):
            a, b = offsets[e], offsets[e + 1]
            if a == b:
                continue
            t = torch.div(s["perm"][a:b].long(), k, rounding_mode="floor")
            gu = torch.mm(q[t], s["gate_up"][e].double().t()) * sc[t] * s["gate_up_scales"][e].double()
            h = gu[:, :I] * torch.sigmoid(gu[:, :I]) * gu[:, I:]
            top = h.abs().amax(1, keepdim=True)
            rows[a:b] = torch.mm((h * (127.0 / top)).round(), s["down"][e].double().t()) * (top / 127.0)
            rows[a:b] *= s["down_scales"][e].double()
        place = s["inv"].long().view(T, k)
        out = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        for j in range(k):
            out += rows[place[:, j]] * s["weights"][:, j:j + 1].double()
        return {"rows": rows, "out": out}
    place, w, g = s["inv"].long().view(T, k), s["weights"].double(), s["grad_out"].double()
    grad_y = torch.empty(T * k, H, dtype=torch.float64, device="cuda")
    grad_hidden = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    grad_w = torch.empty(T, k, dtype=torch.float64, device="cuda")
    for j in range(k):
        grad_y[place[:, j]] = g * w[:, j:j + 1]
        grad_w[:, j] = torch.einsum("th,th->t", g, s["y"][place[:, j]].double())
        grad_hidden += s["grad_rows"][place[:, j]].double()
    # softmax over the selected logits: its Jacobian is diag(w) - w w^T
    jac = torch.diag_embed(w) - w.unsqueeze(2) * w.unsqueeze(1)
    grad_logits = torch.zeros(T, case["E"], dtype=torch.float64, device="cuda")
    grad_logits.scatter_add_(1, s["idx"].long(), torch.einsum("tij,tj->ti", jac, grad_w))
    return {"grad_y": grad_y, "grad_weights": grad_w, "grad_logits": grad_logits, "grad_hidden": grad_hidden}
