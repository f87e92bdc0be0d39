"""Products of experts' layers, measured: tokens grouped by expert times each expert's weights (forward, and the gradient
of the tokens with the weights read the other way), the gradient of the weights (a product over each expert's own tokens),
and products of 8-bit integers with a scale for each token and each channel, for one matrix and for groups.

Matrices are column-major as everywhere in this library: a token is one column, its features contiguous, so that the
tensors below have a token for a row."""
import math

import numpy as np
import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _products(name, type, mode, op, groups, active, n, m, k, out=None):
    return {"name": name, "do": "products", "type": type, "mode": mode, "op": op, "groups": groups, "active": active,
            "n": n, "m": m, "k": k, "out": out or type}


def _weights(name, type, mode, groups, active, k, m, n, out):
    return {"name": name, "do": "weights", "type": type, "mode": mode, "groups": groups, "active": active, "k": k,
            "m": m, "n": n, "out": out}


def _int8(name, type, groups, active, n, m, k, out):
    return {"name": name, "do": "int8", "type": type, "groups": groups, "active": active, "n": n, "m": m, "k": k,
            "out": out}


def listed():
    return [
        # training, a large layer: 16384 tokens of a step to 8 experts
        _products("forward_bf16", "bf16", "", "T", 8, 8, 16384, 4096, 2048),
        # the gradient of the tokens, the same weights read the other way; many smaller experts, one of them idle
        _products("tokens_gradient_bf16", "bf16", "", "N", 16, 15, 8192, 2048, 1536),
        # FP32 training on the matrix cores, error-corrected: what this library does for one product
        _products("forward_f32", "f32", "FP16TCEC", "T", 8, 8, 4096, 2048, 1024),
        # FP32 with the full exponent range, sizes no tile divides
        _products("forward_f32_odd", "f32", "TF32TCEC", "N", 6, 5, 1531, 1021, 777),
        # serving: eight sequences' next tokens, eight experts each
        _products("serve_bf16", "bf16", "", "T", 64, 40, 64, 2048, 1024),
        # one sequence's next token, FP32, two of eight experts: latency
        _products("token_f32", "f32", "FP16TCEC", "T", 8, 2, 2, 1024, 1024),
        # the gradient of the large layer's weights, accumulated and kept in FP32
        _weights("weights_bf16", "bf16", "", 8, 8, 16384, 4096, 2048, "f32"),
        # FP32 weights' gradients, two experts without a token
        _weights("weights_f32", "f32", "FP16TCEC", 16, 14, 4096, 1024, 1024, "f32"),
        # sizes no tile divides and rows that are not aligned to 16 bytes, FP16
        _weights("weights_f16_odd", "f16", "", 5, 5, 1001, 515, 389, "f16"),
        # a prompt of 8192 tokens through one layer in 8-bit integers, activations quantised on the way
        _int8("int8_prompt", "bf16", 1, 1, 8192, 4096, 4096, "bf16"),
        # one token through the same layer
        _int8("int8_token", "bf16", 1, 1, 1, 4096, 4096, "bf16"),
        # experts' layer in 8-bit integers, a batch of 256 tokens
        _int8("int8_experts", "f16", 32, 30, 256, 2048, 1536, "f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _side(rng, lo, hi):
    """A number of features: a multiple of 64, of 8, or any number."""
    v, step = _log(rng, lo, hi), rng.choice([64, 64, 64, 8, 1])
    v = max(step, v // step * step)
    return v + 64 if v == 3072 else v


def draw(rng):
    do = rng.choice(["products", "products", "weights", "int8"])
    groups = _log(rng, 1, 64)
    tokens = _log(rng, 1, 16384)
    active = max(1, min(groups, tokens, int(groups * rng.uniform(0.5, 1.2))))
    m, k = _side(rng, 256, 4096), _side(rng, 256, 2048)
    while groups * m * k > 1 << 28:
        groups = max(1, groups // 2)
    active = min(active, groups)
    type = rng.choice(["f32", "bf16", "f16"])
    mode = rng.choice(["FP16TCEC", "TF32TCEC"]) if type == "f32" else ""
    if do == "int8":
        return _without_name(_int8("", type, groups, active, tokens, m, k, rng.choice(["bf16", "f16"])))
    if type == "f32":  # (FP32 products cost more: as many tokens as keep them below the largest case listed)
        tokens = max(active, tokens // 4)
    if do == "weights":
        out = rng.choice(["f32", type])
        return _without_name(_weights("", type, mode, groups, active, tokens, m, k, out))
    return _without_name(_products("", type, mode, rng.choice(["T", "N"]), groups, active, tokens, m, k))


def _without_name(case):
    return {key: value for key, value in case.items() if key != "name"}


def _tokens_of(case):
    return case["k"] if case["do"] == "weights" else case["n"]


def _sizes(case, seed):
    """How many tokens each group has: `active` of them at least one, some several times as many as others."""
    rng = np.random.RandomState(seed % (1 << 31))
    tokens, active = _tokens_of(case), case["active"]
    share = np.exp(0.4 * rng.randn(active))
    more = np.floor(share / share.sum() * (tokens - active)).astype(np.int64)
    more[: tokens - active - int(more.sum())] += 1
    sizes = np.zeros(case["groups"], np.int64)
    sizes[rng.permutation(case["groups"])[:active]] = 1 + more
    return sizes


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale

    sizes = _sizes(case, seed)
    offsets = torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)).cuda()
    s = {"case": case, "offsets": offsets, "most": int(sizes.max())}
    if case["do"] == "weights":
        dt = DTYPE[case["type"]]
        s["a"] = normal(case["k"], case["m"], scale=0.1).to(dt)  # gradients of the layer's results
        s["b"] = normal(case["k"], case["n"]).to(dt)             # the tokens
        return s
    groups, m, k = case["groups"], case["m"], case["k"]
    s["x"] = normal(case["n"], k).to(DTYPE[case["type"]])
    if case["do"] == "int8":
        w = normal(groups, m, k, scale=k ** -0.5)
        s["w_scale"] = w.abs().amax(2) / 127.0
        s["w"] = torch.round(w / s["w_scale"][..., None]).clamp(-127, 127).to(torch.int8)
    else:
        shape = (groups, m, k) if case["op"] == "T" else (groups, k, m)
        s["w"] = normal(*shape, scale=k ** -0.5).to(DTYPE[case["type"]])
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ---- plain forms ----

def _padded(s):
    """For each group the numbers of its tokens, padded to the largest group's, and which of them are its own."""
    off = s["offsets"].long()
    index = off[:-1, None] + torch.arange(s["most"], device=off.device)[None]
    valid = index < off[1:, None]
    return torch.where(valid, index, 0), valid


def _of_tokens(s, padded):
    """The tokens' rows of padded groups' results."""
    off = s["offsets"].long()
    token = torch.arange(_tokens_of(s["case"]), device=off.device)
    group = torch.searchsorted(off[1:], token, right=True)
    return padded[group, token - off[group]]


def _plain_products(x, w, s):
    """x[token] times its group's w[group] (m rows of k), in 32 bits."""
    if s["case"]["groups"] == 1:
        return x @ w[0].T
    index, valid = _padded(s)
    rows = torch.where(valid[..., None], x[index], 0.0)
    return _of_tokens(s, torch.bmm(rows, w.transpose(1, 2)))


def _plain(s):
    c = s["case"]
    if c["do"] == "weights":
        index, valid = _padded(s)
        a = torch.where(valid[..., None], s["a"].float()[index], 0.0)
        b = torch.where(valid[..., None], s["b"].float()[index], 0.0)
        return torch.bmm(b.transpose(1, 2), a).to(DTYPE[c["out"]])
    x = s["x"].float()
    if c["do"] == "products":
        w = s["w"].float()
        return _plain_products(x, w if c["op"] == "T" else w.transpose(1, 2), s).to(DTYPE[c["out"]])
    scale = x.abs().amax(1) / 127.0
    q = torch.round(x / scale[:, None]).clamp(-127, 127)
    y = _plain_products(q, s["w"].float(), s) * scale[:, None]
    off = s["offsets"].long()
    token = torch.arange(c["n"], device=off.device)
    return (y * s["w_scale"][torch.searchsorted(off[1:], token, right=True)]).to(DTYPE[c["out"]])


# ---- the library's ----

_kept = {}


def _handle():
    if not _kept:
        import cumpsgemm_amd as cg
        _kept["cg"] = cg
        _kept["handle"] = cg.Handle(stream=torch.cuda.current_stream())
        _kept["type"] = {"f32": cg.R_32F, "f16": cg.R_16F, "bf16": cg.R_16BF}
        _kept["mode"] = {"": cg.FP16TC, "FP16TCEC": cg.FP16TCEC, "TF32TCEC": cg.TF32TCEC}
        _kept["op"] = {"T": cg.OP_T, "N": cg.OP_N}
    return _kept["handle"]


def _own(s):
    h, c = _handle(), s["case"]
    m, n, k, groups = c["m"], c["n"], c["k"], c["groups"]
    type, out = _kept["type"][c["type"]], _kept["type"][c["out"]]
    if c["do"] == "weights":
        y = torch.empty(groups, n, m, device="cuda", dtype=DTYPE[c["out"]])
        st = h.gemm_grouped_k(m, n, k, 1.0, s["a"], m, s["b"], n, 0.0, y, m, m * n, s["offsets"], groups,
                              _kept["mode"][c["mode"]], type, out)
    elif c["do"] == "products":
        y = torch.empty(n, m, device="cuda", dtype=DTYPE[c["out"]])
        st = h.gemm_grouped(_kept["op"][c["op"]], m, n, k, 1.0, s["w"], k if c["op"] == "T" else m, m * k, s["x"], k, 0.0,
                            y, m, s["offsets"], groups, _kept["mode"][c["mode"]], type, out)
    else:
        y = torch.empty(n, m, device="cuda", dtype=DTYPE[c["out"]])
        q = torch.empty(n, k, device="cuda", dtype=torch.int8)
        scale = torch.empty(n, device="cuda", dtype=torch.float32)
        st = h.quantize_i8(k, n, s["x"], k, type, q, k, scale)
        if st == 0:
            st = h.gemm_i8(m, n, k, s["w"], k, m * k, s["w_scale"], q, k, scale, y, m, out,
                           s["offsets"] if groups > 1 else None, groups)
    if st != 0:
        raise RuntimeError("status %d" % st)
    return y


def run(s):
    return _own(s) if own else _plain(s)


def exact(case, seed):
    """Group by group in FP64."""
    s = _inputs(case, seed)
    off = s["offsets"].tolist()
    spans = list(zip(off[:-1], off[1:]))
    if case["do"] == "weights":
        a, b = s["a"].double(), s["b"].double()
        return torch.stack([b[lo:hi].t().contiguous() @ a[lo:hi] for lo, hi in spans])
    x = s["x"].double()
    y = torch.empty(case["n"], case["m"], device="cuda", dtype=torch.float64)
    if case["do"] == "int8":
        step = x.abs().max(dim=1, keepdim=True).values / 127
        x = torch.clamp(torch.round(x / step), -127, 127) * step
    for g, (lo, hi) in enumerate(spans):
        w = s["w"][g].double()
        if case["do"] == "int8":
            w = w * s["w_scale"][g].double()[:, None]
        y[lo:hi] = x[lo:hi] @ (w if case.get("op") == "N" else w.t().contiguous())
    return y


def work(case):
    active, tokens = case["active"], _tokens_of(case)
    es, out = BYTES[case["type"]], BYTES[case["out"]]
    m, other = case["m"], case["n"] if case["do"] == "weights" else case["k"]
    flops = 2 * tokens * m * other
    if case["do"] == "weights":
        return {"bytes": tokens * (m + other) * es + case["groups"] * m * other * out, "flops": flops}
    if case["do"] == "int8":
        return {"bytes": tokens * other * es + active * m * (other + 4) + tokens * m * out, "flops": flops}
    return {"bytes": tokens * other * es + active * m * other * es + tokens * m * out, "flops": flops}
