"""Gated feed-forward blocks and products in 8-bit floating point, measured: both projections of a block with their activation
and product (forward; with the projections kept, for training), the gradient that comes back through them, products of FP8
values with a scale for each block of 128, either way through the weights, and the gated block served in FP8.  Dense (one
group) and for tokens grouped by expert.

Matrices are column-major as everywhere in this library: a token is one column, its features contiguous, so that the
tensors below have a token for a row."""
import math

import numpy as np
import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn,
         "e5m2": torch.float8_e5m2}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "e5m2": 1}
MOST = {"e4m3": 448.0, "e5m2": 57344.0}


def _gated(name, type, mode, op, act, keep, groups, active, n, m, k):
    return {"name": name, "do": "gated", "type": type, "mode": mode, "op": op, "act": act, "keep": keep, "groups": groups,
            "active": active, "n": n, "m": m, "k": k}


def _backward(name, type, mode, op, act, groups, active, n, m, k):
    return {"name": name, "do": "backward", "type": type, "mode": mode, "op": op, "act": act, "groups": groups,
            "active": active, "n": n, "m": m, "k": k}


def _f8(name, type, f8, op, groups, active, n, m, k):
    return {"name": name, "do": "f8", "type": type, "f8": f8, "op": op, "groups": groups, "active": active, "n": n, "m": m,
            "k": k}


def _block_f8(name, type, act, groups, active, n, m, k):
    return {"name": name, "do": "block_f8", "type": type, "act": act, "groups": groups, "active": active, "n": n, "m": m,
            "k": k}


def listed():
    return [
        # training, a large layer of experts: 16384 tokens of a step to 8 gated experts, the projections kept
        _gated("gated_bf16", "bf16", "", "T", "silu", True, 8, 8, 16384, 2048, 2048),
        # FP32 training on the matrix cores, error-corrected; many smaller experts, two of them idle
        _gated("gated_f32", "f32", "FP16TCEC", "T", "gelu", True, 16, 14, 4096, 1024, 1024),
        # sizes no tile divides, rows of no alignment, weights stored the other way round
        _gated("gated_f16_odd", "f16", "", "N", "gelu_tanh", False, 5, 5, 1001, 515, 389),
        # one sequence's next token through a dense block: latency
        _gated("gated_token_bf16", "bf16", "", "T", "silu", False, 1, 1, 1, 4096, 2048),
        # the gradient of the large layer's projections
        _backward("backward_bf16", "bf16", "", "N", "silu", 8, 8, 16384, 2048, 2048),
        # ... of the FP32 layer's, with FP32's range
        _backward("backward_f32", "f32", "TF32TCEC", "N", "gelu", 16, 14, 4096, 1024, 1024),
        # ... at sizes no tile divides
        _backward("backward_f16_odd", "f16", "", "N", "gelu_tanh", 5, 5, 1001, 515, 389),
        # a prompt of 8192 tokens through one layer in FP8, activations quantised on the way
        _f8("f8_prompt", "bf16", "e4m3", "T", 1, 1, 8192, 4096, 4096),
        # one token through the same layer
        _f8("f8_token", "bf16", "e4m3", "T", 1, 1, 1, 4096, 4096),
        # FP8 training: gradients of 1531 tokens in E5M2 back through experts' weights that are kept as the forward pass has them
        _f8("f8_gradient", "bf16", "e5m2", "N", 8, 7, 1531, 2048, 1536),
        # gated experts served in FP8, a prompt of 4096 tokens: projections, activation and the product behind them
        _block_f8("block_f8_prompt", "bf16", "silu", 8, 8, 4096, 2048, 2048),
        # a batch of eight sequences' next tokens, eight experts each
        _block_f8("block_f8_tokens", "bf16", "silu", 64, 40, 64, 1024, 2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _side(rng, lo, hi):
    """A number of features: a multiple of 128, of 16, or any number."""
    v, step = _log(rng, lo, hi), rng.choice([128, 128, 128, 16, 1])
    return max(step, v // step * step)


def draw(rng):
    do = rng.choice(["gated", "backward", "f8", "block_f8"])
    groups = _log(rng, 1, 64)
    tokens = _log(rng, 1, 16384)
    m, k = _side(rng, 256, 4096), _side(rng, 256, 2048)
    while groups * m * k > 1 << 27:
        groups = max(1, groups // 2)
    type = rng.choice(["f32", "bf16", "f16"])
    mode = rng.choice(["FP16TCEC", "TF32TCEC"]) if type == "f32" else ""
    # (no more work than the largest cases listed; FP32 products cost more)
    products = {"gated": 2, "backward": 1, "f8": 1, "block_f8": 3}[do]
    while products * tokens * m * k > (1 << 33 if type == "f32" and not do.endswith("f8") else 1 << 36):
        tokens = max(1, tokens // 2)
    active = max(1, min(groups, tokens, int(groups * rng.uniform(0.5, 1.2))))
    act, op = rng.choice(["silu", "gelu", "gelu_tanh", "relu"]), rng.choice(["T", "N"])
    if do == "gated":
        case = _gated("", type, mode, op, act, rng.choice([True, False]), groups, active, tokens, m, k)
    elif do == "backward":
        case = _backward("", type, mode, op, act, groups, active, tokens, m, k)
    elif do == "f8":
        case = _f8("", rng.choice(["bf16", "f16"]), rng.choice(["e4m3", "e5m2"]), op, groups, active, tokens, m, k)
    else:
        case = _block_f8("", rng.choice(["bf16", "f16"]), act, groups, active, tokens, m, k)
    return {key: value for key, value in case.items() if key != "name"}


def _sizes(case, seed):
    """How many tokens each group has: `active` of them at least one, some several times as many as others."""
    rng = np.random.RandomState(seed % (1 << 31))
    tokens, active = case["n"], case["active"]
    share = np.exp(0.4 * rng.randn(active))
    more = np.floor(share / share.sum() * (tokens - active)).astype(np.int64)
    more[: tokens - active - int(more.sum())] += 1
    sizes = np.zeros(case["groups"], np.int64)
    sizes[rng.permutation(case["groups"])[:active]] = 1 + more
    return sizes


def _blocks(size):
    return (size + 127) // 128


def _weights_f8(w, f8):
    """[groups, rows, cols] in FP8 with a scale for each 128 x 128: (values, [groups, row blocks, column blocks])."""
    groups, rows, cols = w.shape
    rb, cb = _blocks(rows), _blocks(cols)
    full = torch.zeros(groups, rb * 128, cb * 128, device=w.device)
    full[:, :rows, :cols] = w
    full = full.view(groups, rb, 128, cb, 128)
    peak = full.abs().amax((2, 4))
    q = (full * MOST[f8] / peak[:, :, None, :, None]).to(DTYPE[f8]).view(groups, rb * 128, cb * 128)
    return q[:, :rows, :cols].contiguous(), peak / MOST[f8]


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale

    sizes = _sizes(case, seed)
    offsets = torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)).cuda()
    s = {"case": case, "offsets": offsets, "most": int(sizes.max())}
    do, groups, n, m, k = case["do"], case["groups"], case["n"], case["m"], case["k"]
    dt = DTYPE[case["type"]]
    if do == "gated":
        shape = (2, groups, m, k) if case["op"] == "T" else (2, groups, k, m)  # gate, up
        s["w"] = normal(*shape, scale=k ** -0.5).to(dt)
        s["x"] = normal(n, k).to(dt)
    elif do == "backward":
        s["w"] = normal(*((groups, m, k) if case["op"] == "T" else (groups, k, m)), scale=k ** -0.5).to(dt)
        s["dy"] = normal(n, k, scale=0.1).to(dt)
        s["z"] = normal(2, n, m).to(dt)
    elif do == "f8":
        shape = (groups, m, k) if case["op"] == "T" else (groups, k, m)
        s["w"], s["w_scale"] = _weights_f8(normal(*shape, scale=k ** -0.5), "e4m3")
        s["x"] = normal(n, k, scale=1.0 if case["f8"] == "e4m3" else 0.01).to(dt)
    else:
        s["gate"], s["gate_scale"] = _weights_f8(normal(groups, m, k, scale=k ** -0.5), "e4m3")
        s["up"], s["up_scale"] = _weights_f8(normal(groups, m, k, scale=k ** -0.5), "e4m3")
        s["down"], s["down_scale"] = _weights_f8(normal(groups, k, m, scale=m ** -0.5), "e4m3")
        s["x"] = normal(n, k).to(dt)
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ---- plain forms ----

def _product(x, w, s):
    """x[token] times its group's w[group] (m rows of k), in 32 bits."""
    if s["case"]["groups"] == 1:
        return x @ w[0].T
    off = s["offsets"].long()
    index = off[:-1, None] + torch.arange(s["most"], device=off.device)[None]
    valid = index < off[1:, None]
    rows = torch.where(valid[..., None], x[torch.where(valid, index, 0)], 0.0)
    y = torch.bmm(rows, w.transpose(1, 2))
    token = torch.arange(s["case"]["n"], device=off.device)
    group = torch.searchsorted(off[1:], token, right=True)
    return y[group, token - off[group]]


def _activation(act, g):
    """act(g) and its derivative, in g's own type."""
    if act == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if act == "gelu":
        # the distribution function of a normal variable, and its density
        below = 0.5 * torch.erfc(g * -math.sqrt(0.5))
        return g * below, below + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s + g * s * (1 - s)
    c = 2 * math.sqrt(2 / math.pi)
    s = 1 / (1 + torch.exp(-c * (g + 0.044715 * g * g * g)))
    return g * s, s + g * s * (1 - s) * c * (1 + 3 * 0.044715 * g * g)


def _quantised(x, f8):
    """Each token's values in FP8 with a scale for each 128, as the values that they stand for."""
    n, k = x.shape
    full = torch.zeros(n, _blocks(k) * 128, device=x.device)
    full[:, :k] = x
    full = full.view(n, -1, 128)
    peak = full.abs().amax(2, keepdim=True)
    # (MOST x is exact for 16-bit x, and so is a quotient half way between two FP8 values, where such x often lead)
    q = (full * MOST[f8] / peak).to(DTYPE[f8]).float()
    return torch.where(peak > 0, q * (peak / MOST[f8]), 0.0).view(n, -1)[:, :k]


def _values(q, scale):
    """Weights in FP8 as the values that they stand for."""
    return q.float() * scale.repeat_interleave(128, 1).repeat_interleave(128, 2)[:, :q.shape[1], :q.shape[2]]


def _plain(s):
    c = s["case"]
    dt = DTYPE[c["type"]]
    if c["do"] == "gated":
        w = s["w"].float() if c["op"] == "T" else s["w"].float().transpose(2, 3)
        gate, up = _product(s["x"].float(), w[0], s), _product(s["x"].float(), w[1], s)
        h = _activation(c["act"], gate)[0] * up
        return (h.to(dt), gate.to(dt), up.to(dt)) if c["keep"] else h.to(dt)
    if c["do"] == "backward":
        w = s["w"].float() if c["op"] == "T" else s["w"].float().transpose(1, 2)
        dh = _product(s["dy"].float(), w, s)
        gate, up = s["z"].float()
        a, da = _activation(c["act"], gate)
        return (dh * up * da).to(dt), (dh * a).to(dt), (a * up).to(dt)
    if c["do"] == "f8":
        w = _values(s["w"], s["w_scale"])
        return _product(_quantised(s["x"].float(), c["f8"]), w if c["op"] == "T" else w.transpose(1, 2), s).to(dt)
    x = _quantised(s["x"].float(), "e4m3")
    gate, up = _product(x, _values(s["gate"], s["gate_scale"]), s), _product(x, _values(s["up"], s["up_scale"]), s)
    h = (_activation(c["act"], gate)[0] * up).to(dt).float()
    return _product(_quantised(h, "e4m3"), _values(s["down"], s["down_scale"]), s).to(dt)


# ---- the library's ----

_kept = {}


def _handle():
    if not _kept:
        import cumpsgemm_amd as cg
        _kept["handle"] = cg.Handle(stream=torch.cuda.current_stream())
        _kept["type"] = {"f32": cg.R_32F, "f16": cg.R_16F, "bf16": cg.R_16BF, "e4m3": cg.R_8F_E4M3, "e5m2": cg.R_8F_E5M2}
        _kept["mode"] = {"": cg.FP16TC, "FP16TCEC": cg.FP16TCEC, "TF32TCEC": cg.TF32TCEC}
        _kept["op"] = {"T": cg.OP_T, "N": cg.OP_N}
        _kept["act"] = {"silu": cg.SILU, "gelu": cg.GELU, "gelu_tanh": cg.GELU_TANH, "relu": cg.RELU}
    return _kept["handle"]


def _checked(status):
    if status != 0:
        raise RuntimeError("status %d" % status)


def _own_quantised(h, x, n, k, type, f8):
    q = torch.empty(n, k, device="cuda", dtype=DTYPE[f8])
    scale = torch.empty(n, _blocks(k), device="cuda", dtype=torch.float32)
    _checked(h.quantize_f8(k, n, x, k, 0, _kept["type"][type], 1, q, k, 0, _kept["type"][f8], scale))
    return q, scale


def _own(s):
    h, c = _handle(), s["case"]
    do, n, m, k, groups = c["do"], c["n"], c["m"], c["k"], c["groups"]
    type, dt, f8 = _kept["type"][c["type"]], DTYPE[c["type"]], _kept["type"]["e4m3"]
    offsets = s["offsets"] if groups > 1 else None
    if do == "gated":
        y = torch.empty(n, m, device="cuda", dtype=dt)
        z = torch.empty(2, n, m, device="cuda", dtype=dt) if c["keep"] else (None, None)
        _checked(h.gemm_gated(_kept["op"][c["op"]], _kept["act"][c["act"]], m, n, k, s["w"][0], s["w"][1],
                              k if c["op"] == "T" else m, m * k, s["x"], k, y, m, z[0], z[1], m, offsets, groups,
                              _kept["mode"][c["mode"]], type))
        return (y, z[0], z[1]) if c["keep"] else y
    if do == "backward":
        d = torch.empty(3, n, m, device="cuda", dtype=dt)
        _checked(h.gemm_gated_backward(_kept["op"][c["op"]], _kept["act"][c["act"]], m, n, k, s["w"],
                                       k if c["op"] == "T" else m, m * k, s["dy"], k, s["z"][0], s["z"][1], m, d[0], d[1], m,
                                       d[2], m, offsets, groups, _kept["mode"][c["mode"]], type))
        return d[0], d[1], d[2]
    x, x_scale = _own_quantised(h, s["x"], n, k, c["type"], "e4m3" if do == "block_f8" else c["f8"])
    if do == "f8":
        y = torch.empty(n, m, device="cuda", dtype=dt)
        _checked(h.gemm_f8(_kept["op"][c["op"]], m, n, k, s["w"], k if c["op"] == "T" else m, m * k, f8, s["w_scale"],
                           _blocks(m) * _blocks(k), x, k, _kept["type"][c["f8"]], x_scale, y, m, type, offsets, groups))
        return y
    mid = torch.empty(n, m, device="cuda", dtype=dt)
    scales = _blocks(m) * _blocks(k)
    _checked(h.gemm_gated_f8(_kept["act"][c["act"]], m, n, k, s["gate"], s["up"], k, m * k, f8, s["gate_scale"], s["up_scale"],
                             scales, x, k, f8, x_scale, mid, m, type, offsets, groups))
    q, q_scale = _own_quantised(h, mid, n, m, c["type"], "e4m3")
    y = torch.empty(n, k, device="cuda", dtype=dt)
    _checked(h.gemm_f8(_kept["op"]["T"], k, n, m, s["down"], m, m * k, f8, s["down_scale"], scales, q, m, f8, q_scale, y, k,
                       type, offsets, groups))
    return y


def run(s):
    return _own(s) if own else _plain(s)


# ---- in 64 bits ----

def _exact_f8(x, f8):
    """Rounded to FP8 blocks of 128 along the rows, from the format: 4 or 3 significant bits, exponents from -6 or -14 on."""
    bits, least = (4, -6) if f8 == "e4m3" else (3, -14)
    out = torch.zeros_like(x)
    for at in range(0, x.shape[1], 128):
        part = x[:, at:at + 128]
        peak = part.abs().max(dim=1, keepdim=True).values
        v = part * MOST[f8] / peak
        step = torch.exp2((torch.frexp(v)[1] - 1).clamp(min=least).double() - (bits - 1))
        out[:, at:at + 128] = torch.where(peak > 0, torch.round(v / step) * step * (peak / MOST[f8]), 0.0)
    return out


def _exact_weights(q, scale):
    w = q.to(torch.float64)
    for i in range(scale.shape[0]):
        for j in range(scale.shape[1]):
            w[i * 128:i * 128 + 128, j * 128:j * 128 + 128] *= scale[i, j].double()
    return w


def _exact_act(act, g):
    """The activation and, by the formula, its derivative."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        p = torch.special.ndtr(g)
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * g * g)
    return torch.clamp(g, min=0), torch.where(g > 0, 1.0, 0.0).double()


def exact(case, seed):
    """Group by group in FP64."""
    s = _inputs(case, seed)
    off = s["offsets"].tolist()
    spans = [(g, lo, hi) for g, (lo, hi) in enumerate(zip(off[:-1], off[1:])) if hi > lo]
    do, n, m, k = case["do"], case["n"], case["m"], case["k"]

    def side(w):  # [rows of k]
        return w.double() if do == "block_f8" or case["op"] == "T" else w.double().t().contiguous()

    def rows():
        return torch.empty(n, m, device="cuda", dtype=torch.float64)

    if do == "gated":
        gate, up, x = rows(), rows(), s["x"].double()
        for g, lo, hi in spans:
            gate[lo:hi], up[lo:hi] = x[lo:hi] @ side(s["w"][0, g]).t(), x[lo:hi] @ side(s["w"][1, g]).t()
        h = _exact_act(case["act"], gate)[0] * up
        return (h, gate, up) if case["keep"] else h
    if do == "backward":
        dh, dy = rows(), s["dy"].double()
        for g, lo, hi in spans:
            dh[lo:hi] = dy[lo:hi] @ side(s["w"][g]).t()
        gate, up = s["z"].double()
        a, da = _exact_act(case["act"], gate)
        return dh * up * da, dh * a, a * up
    if do == "f8":
        y, x = rows(), _exact_f8(s["x"].double(), case["f8"])
        for g, lo, hi in spans:
            y[lo:hi] = x[lo:hi] @ side(_exact_weights(s["w"][g], s["w_scale"][g])).t()
        return y
    gate, up, x = rows(), rows(), _exact_f8(s["x"].double(), "e4m3")
    for g, lo, hi in spans:
        gate[lo:hi] = x[lo:hi] @ _exact_weights(s["gate"][g], s["gate_scale"][g]).t()
        up[lo:hi] = x[lo:hi] @ _exact_weights(s["up"][g], s["up_scale"][g]).t()
    h = _exact_f8((_exact_act(case["act"], gate)[0] * up).to(DTYPE[case["type"]]).double(), "e4m3")
    y = torch.empty(n, k, device="cuda", dtype=torch.float64)
    for g, lo, hi in spans:
        y[lo:hi] = h[lo:hi] @ _exact_weights(s["down"][g], s["down_scale"][g]).t()
    return y


def work(case):
    do, n, m, k, active, es = case["do"], case["n"], case["m"], case["k"], case["active"], BYTES[case["type"]]
    if do == "gated":
        out = 3 if case["keep"] else 1
        return {"bytes": n * k * es + 2 * active * m * k * es + out * n * m * es, "flops": 4 * n * m * k}
    if do == "backward":
        return {"bytes": n * k * es + active * m * k * es + 5 * n * m * es, "flops": 2 * n * m * k}
    scales = 4 * _blocks(m) * _blocks(k)
    if do == "f8":
        return {"bytes": n * k * es + active * (m * k + scales) + n * m * es, "flops": 2 * n * m * k}
    return {"bytes": 2 * n * k * es + 3 * active * (m * k + scales), "flops": 6 * n * m * k}
