"""Cases of the 8-bit linear path and of the token scores: RMSNorm with the residual's addition and an 8-bit result, row
quantisation (plain and behind SiLU * up), the linear on 8-bit integers, and log probabilities of given tokens with entropy, top
alternatives and gradient.

`run` computes a case in its plain form (elementary torch operations in 32 bits) or, where `own` is true, through the
framework's entry points on buffers that the caller keeps.  What is held in 8 bits is returned as the BF16 values it stands for.
Widths follow the decoder of this repository (hidden 4096, feed-forward 14336, vocabulary 32000) and generic larger ones."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IGNORE = -100
SMALLEST_SCALE = 2.0 ** -126


def listed():
    return [
        # one decoded token between two blocks of the decoder: latency alone
        {"name": "norm 1 token", "op": "norm", "rows": 1, "width": 4096, "residual": True, "type": "bf16"},
        # a prefill of 8192 tokens
        {"name": "norm 8192 tokens", "op": "norm", "rows": 8192, "width": 4096, "residual": True, "type": "bf16"},
        # the activation in front of the down projection, gate and up as the two halves of one projection's output
        {"name": "silu 4096 tokens", "op": "quantize", "rows": 4096, "width": 14336, "gated": True, "type": "bf16"},
        # FP32 rows of an odd width (a projection of an unaligned model, or weights being prepared)
        {"name": "rows of odd width", "op": "quantize", "rows": 1777, "width": 5003, "gated": False, "type": "f32"},
        # the query/key/value projection of one decoded token: the weights are read once
        {"name": "linear 1 token", "op": "linear", "m": 1, "n": 6144, "k": 4096, "bias": False, "type": "bf16"},
        # the down projection of a small decoding batch
        {"name": "linear 17 tokens", "op": "linear", "m": 17, "n": 4096, "k": 14336, "bias": False, "type": "bf16"},
        # ragged sizes with bias and FP32 result
        {"name": "linear ragged", "op": "linear", "m": 1003, "n": 5001, "k": 4112, "bias": True, "type": "f32"},
        # the up projection of a prefill
        {"name": "linear 4096 tokens", "op": "linear", "m": 4096, "n": 14336, "k": 4096, "bias": False, "type": "bf16"},
        # answering with alternatives: a few rows over a large vocabulary
        {"name": "score 4 rows top 20", "op": "score", "rows": 4, "vocab": 128000, "pad": 0, "top": 20, "type": "bf16"},
        # scoring a prompt: FP32 logits of a vocabulary stored with padding behind each row
        {"name": "score 2048 rows top 5", "op": "score", "rows": 2048, "vocab": 32000, "pad": 64, "top": 5, "type": "f32"},
        # a policy-gradient step: log probability and entropy with the logits' gradient
        {"name": "train 2048 rows", "op": "train", "rows": 2048, "vocab": 128000, "pad": 0, "type": "bf16"},
        # the same for a small batch over an odd vocabulary in FP32
        {"name": "train odd vocabulary", "op": "train", "rows": 500, "vocab": 32003, "pad": 0, "type": "f32"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "linear", "score", "train"])
    if op == "norm":
        width = 4 * _log(rng, 64, 4096)
        return {"op": op, "rows": min(_log(rng, 1, 8192), 8192 * 4096 // width), "width": width, "residual": rng.random() < 0.7,
                "type": rng.choice(["bf16", "bf16", "f32"])}
    if op == "quantize":
        width = _log(rng, 128, 20000)
        return {"op": op, "rows": min(_log(rng, 1, 8192), 4096 * 14336 // width), "width": width, "gated": rng.random() < 0.6,
                "type": rng.choice(["bf16", "bf16", "f32", "f16"])}
    if op == "linear":
        n, k = _log(rng, 128, 14336), 16 * _log(rng, 8, 896)
        return {"op": op, "m": min(_log(rng, 1, 4096), 4096 * 14336 * 4096 // (n * k)), "n": n, "k": k, "bias": rng.random() < 0.3,
                "type": rng.choice(["bf16", "bf16", "f32", "f16"])}
    vocab = _log(rng, 1000, 150000)
    case = {"op": op, "rows": min(_log(rng, 1, 2048), 2048 * 32000 // vocab if op == "score" else 2048 * 100000 // vocab), "vocab": vocab, "pad": rng.choice([0, 0, 1, 61]),
            "type": rng.choice(["bf16", "bf16", "f32", "f16"])}
    return {**case, "top": rng.randint(0, 32)} if op == "score" else case


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")
    t = TYPES[case["type"]]
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        channel = torch.where(torch.rand(width, generator=g, device="cuda") < 0.01, 8.0, 1.0)   # the few channels that stand out in a residual stream
        return {"x": (normal(rows, width) * channel).to(t), "delta": (normal(rows, width) * 0.5).to(t) if case["residual"] else None,
                "weight": (1 + 0.1 * normal(width)).to(t), "eps": 1e-5}
    if case["op"] == "quantize":
        rows, width = case["rows"], case["width"]
        if not case["gated"]:
            return {"x": normal(rows, width).to(t), "up": None}
        both = normal(rows, 2 * width).to(t)               # the fused gate and up projection's output, read in place
        return {"x": both[:, :width], "up": both[:, width:]}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]

        def whole(rows):
            return (normal(rows, k) * 32).round().clamp(-127, 127).to(torch.int8)
        return {"x": whole(m), "sx": 0.01 + 0.02 * torch.rand(m, generator=g, device="cuda"), "w": whole(n),
                "sw": 0.0002 + 0.0004 * torch.rand(n, generator=g, device="cuda"), "bias": normal(n) if case["bias"] else None, "type": t}
    rows, vocab, pad = case["rows"], case["vocab"], case["pad"]
    logits = torch.empty(rows, vocab + pad, device="cuda", dtype=t)
    for at in range(0, rows, 256):
        logits[at:at + 256] = (normal(min(256, rows - at), vocab + pad) * 2.5).to(t)
    logits = logits[:, :vocab]
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    ids = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.1, IGNORE, ids)   # prompt and padding positions are not scored
    # half of the scored tokens are the likeliest one, as in a model's own samples
    best = logits.float().argmax(-1)
    ids = torch.where((ids != IGNORE) & (torch.rand(rows, generator=g, device="cuda") < 0.5), best, ids)
    state = {"logits": logits, "ids": ids, "scale": 1.25}                                 # sampling temperature 0.8
    if case["op"] == "train":
        state |= {"g_log_prob": normal(rows) / rows, "g_entropy": torch.full((rows,), 0.01 / rows, device="cuda")}
    return state


def prepare(case, seed):
    state = {"op": case["op"], "case": case, **_inputs(case, seed)}
    if own:
        _bind(state)
    return state


# ---- the framework's calls ---------------------------------------------------------------------------------------------
class _Handles:
    """The framework's descriptors of torch tensors; the registrations end with it."""

    def __init__(self):
        from rust_ascend_b200 import B200Runtime, DType, RuntimeOptions
        if B200Runtime._ctx is None:
            B200Runtime.initialize_exclusive(RuntimeOptions(device=0))
        self.client = B200Runtime.client(B200Runtime._device)
        self.types = {torch.float32: DType.F32, torch.bfloat16: DType.BF16, torch.float16: DType.F16, torch.int8: DType.I8, torch.int32: DType.I32, torch.int64: DType.I64}
        self.handles = []

    def __call__(self, t):
        from rust_ascend_b200 import TensorBuffer
        if t is None:
            return None
        whole = t.untyped_storage()
        self.handles.append(self.client.import_pointer(whole.data_ptr(), whole.nbytes()))
        return TensorBuffer(self.handles[-1], tuple(t.shape), self.types[t.dtype], tuple(t.stride()), t.storage_offset() * t.element_size())

    def __del__(self):
        for h in self.handles:
            self.client.free(h)


def _bind(state):
    """The buffers that the caller keeps: results, and descriptors of everything the calls read or write."""
    h = state["handles"] = _Handles()
    op, case = state["op"], state["case"]

    def new(dtype, *shape):
        return torch.empty(shape, device="cuda", dtype=dtype)
    if op in ("norm", "quantize"):
        rows, width = case["rows"], case["width"]
        q, scales, values = new(torch.int8, rows, width), new(torch.float32, rows), new(torch.bfloat16, rows, width)
        total = torch.empty_like(state["x"]) if state.get("delta") is not None else None
        state["out"] = {"values": values, "scales": scales} | ({"total": total} if total is not None else {})
        state["kept"] = q
        state["b"] = {"x": h(state["x"]), "q": h(q), "scales": h(scales), "values": h(values), "total": h(total), "delta": h(state.get("delta")),
                      "weight": h(state.get("weight")), "up": h(state.get("up"))}
    elif op == "linear":
        y = new(state["type"], case["m"], case["n"])
        state["out"] = y
        state["b"] = {"y": h(y)} | {k: h(state[k]) for k in ("x", "sx", "w", "sw", "bias")}
    else:
        rows, top = case["rows"], case.get("top", 0)
        out = {k: new(torch.float32, rows) for k in ("log_prob", "lse", "entropy")}
        if top:
            out |= {"top_values": new(torch.float32, rows, top), "top_ids": new(torch.int32, rows, top)}
        if op == "train":
            out["d_logits"] = new(state["logits"].dtype, rows, case["vocab"])
        state["out"] = out
        state["b"] = {k: h(v) for k, v in out.items()} | {k: h(state[k]) for k in ("logits", "ids", "g_log_prob", "g_entropy") if k in state}


def _run_own(state):
    from rust_ascend_b200 import B200Runtime as RT
    op, b, c = state["op"], state["b"], state["handles"].client
    if op == "norm":
        RT.rms_norm_quant(c, b["x"], b["weight"], state["eps"], delta=b["delta"], out=(b["q"], b["scales"], b["total"]))
        RT.dequantize_rows(c, b["q"], b["scales"], out=b["values"])
    elif op == "quantize":
        RT.quantize_rows(c, b["x"], up=b["up"], out=(b["q"], b["scales"]))
        RT.dequantize_rows(c, b["q"], b["scales"], out=b["values"])
    elif op == "linear":
        RT.linear_i8(c, b["x"], b["sx"], b["w"], b["sw"], bias=b["bias"], out=b["y"])
    else:
        RT.token_log_probs(c, b["logits"], b["ids"], scale=state["scale"], ignore_index=IGNORE, top_k=state["case"].get("top", 0),
                           out=(b["log_prob"], b["lse"], b["entropy"], b.get("top_values"), b.get("top_ids")))
        if op == "train":
            RT.token_log_probs_backward(c, b["logits"], b["ids"], b["lse"], b["entropy"], b["g_log_prob"], b["g_entropy"], scale=state["scale"],
                                        ignore_index=IGNORE, out=b["d_logits"])
    return state["out"]


# ---- the plain form ----------------------------------------------------------------------------------------------------
def _quantized(y):
    """Symmetric 8-bit rows: values as held, and the scale of each row."""
    scale = (y.abs().amax(-1, keepdim=True) / 127).clamp_min(SMALLEST_SCALE)
    q = (y / scale).round()
    return {"values": (q * scale).to(torch.bfloat16), "scales": scale[:, 0]}


def _plain_score(state):
    z = state["logits"].float() * state["scale"]
    ids, rows = state["ids"], state["logits"].shape[0]
    most = z.amax(-1, keepdim=True)
    lse = most[:, 0] + (z - most).exp().sum(-1).log()
    lp = z - lse[:, None]
    scored = ids != IGNORE
    at = torch.where(scored, ids, 0)
    log_prob = torch.where(scored, lp[torch.arange(rows, device="cuda"), at], 0.0)
    p = lp.exp()
    entropy = -(p * lp).sum(-1)
    out = {"log_prob": log_prob, "lse": lse, "entropy": entropy}
    top = state["case"].get("top", 0)
    if top:
        order = state["logits"].float().sort(dim=-1, descending=True, stable=True)[1][:, :top]
        out |= {"top_values": lp.gather(1, order), "top_ids": order.to(torch.int32)}
    if state["op"] == "train":
        g = torch.where(scored, state["g_log_prob"], 0.0)
        d = -p * (g[:, None] + state["g_entropy"][:, None] * (lp + entropy[:, None]))
        d[torch.arange(rows, device="cuda"), at] += g
        out["d_logits"] = (d * state["scale"]).to(state["logits"].dtype)
    return out


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "norm":
        x, out = state["x"], {}
        if state["delta"] is not None:
            x = (x.float() + state["delta"].float()).to(x.dtype)
            out["total"] = x
        f = x.float()
        y = f * (1 / (f.square().mean(-1, keepdim=True) + state["eps"]).sqrt()) * state["weight"].float()
        return out | _quantized(y)
    if op == "quantize":
        y = state["x"].float()
        if state["up"] is not None:
            y = y / (1 + (-y).exp()) * state["up"].float()
        return _quantized(y)
    if op == "linear":
        y = state["x"].float() @ state["w"].float().T * (state["sx"][:, None] * state["sw"][None, :])
        return (y + state["bias"] if state["bias"] is not None else y).to(state["type"])
    return _plain_score(state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    op, size = case["op"], TYPES[case["type"]].itemsize
    if op == "norm":
        rows, width = case["rows"], case["width"]
        moved = size + (2 * size if case["residual"] else 0) + 2          # x; delta and the sum; the values in BF16
        return {"bytes": rows * (width * moved + 4) + width * size, "flops": 8 * rows * width}
    if op == "quantize":
        rows, width = case["rows"], case["width"]
        return {"bytes": rows * (width * ((2 if case["gated"] else 1) * size + 2) + 4), "flops": 8 * rows * width}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n + (n if case["bias"] else 0)) + m * n * size, "flops": 2 * m * n * k}
    rows, vocab = case["rows"], case["vocab"]
    read, written = rows * (vocab * size + 8), rows * 4 * 3 + rows * 8 * case.get("top", 0)
    if op == "train":
        read, written = read + rows * 8, written + rows * vocab * size
    return {"bytes": read + written, "flops": rows * vocab * (6 if op == "score" else 14)}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "linear":
        acc = torch.matmul(s["x"].double(), s["w"].double().transpose(0, 1))
        acc.mul_(s["sx"].double().unsqueeze(1)).mul_(s["sw"].double())
        return acc if s["bias"] is None else acc + s["bias"].double()
    if case["op"] in ("norm", "quantize"):
        found = {}
        v = s["x"].double()
        if case["op"] == "norm":
            if s["delta"] is not None:
                v = (v + s["delta"].double()).to(s["x"].dtype).double()
                found["total"] = v
            v = v * s["weight"].double() / torch.sqrt((v * v).sum(1, keepdim=True) / case["width"] + s["eps"])
        elif s["up"] is not None:
            v = v * torch.sigmoid(v) * s["up"].double()
        step = torch.clamp(torch.max(torch.abs(v), dim=1).values / 127.0, min=SMALLEST_SCALE)
        found["scales"] = step
        found["values"] = torch.round(v / step.unsqueeze(1)) * step.unsqueeze(1)
        return found
    found = {"log_prob": [], "lse": [], "entropy": []} | ({"d_logits": []} if case["op"] == "train" else {}) | ({"top_values": []} if case.get("top") else {})
    for at in range(0, case["rows"], 256):                       # in blocks of rows: a whole batch in 64 bits is large
        z = s["logits"][at:at + 256].double() * s["scale"]
        ids = s["ids"][at:at + 256]
        lse = torch.logsumexp(z, dim=1)
        lp = torch.log_softmax(z, dim=1)
        p = torch.softmax(z, dim=1)
        entropy = torch.special.entr(p).sum(dim=1)
        live = (ids >= 0).double()
        found["log_prob"].append(lp.gather(1, ids.clamp(min=0).unsqueeze(1)).squeeze(1) * live)
        found["lse"].append(lse)
        found["entropy"].append(entropy)
        if case.get("top"):
            found["top_values"].append(lp.topk(case["top"], dim=1).values)
        if case["op"] == "train":
            up = s["g_log_prob"][at:at + 256].double() * live
            hot = torch.zeros_like(p).scatter_(1, ids.clamp(min=0).unsqueeze(1), 1.0)
            ge = s["g_entropy"][at:at + 256].double().unsqueeze(1)
            # -p (log p + H) is the entropy's gradient; p log p -> 0 with p
            d = up.unsqueeze(1) * (hot - p) + ge * (torch.special.entr(p) - p * entropy.unsqueeze(1))
            found["d_logits"].append(d * s["scale"])
    return {k: torch.cat(v) for k, v in found.items()}
