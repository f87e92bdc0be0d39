"""Gated feed-forward blocks on the library's products, dense (one expert) or of experts: each token goes through the block of
its expert.

    python -m cumpsgemm_amd.gated [tokens [features_in [features [experts]]]]

runs a training step in FP32 on split operands and in BF16 (forward, the gradients of tokens and matrices), then serves the
matrices in 8-bit floating point, and prints how far each result is from FP64.

Tensors hold a token in a row, as in cumpsgemm_amd.experts; all work goes to torch's current stream, whichever the handle has."""
import sys

from . import _lib as lib
from .experts import (_blocks, _check, _expect, _f8_matrices, _matrices_to_f8, _on_current_stream, _sizes, _tokens_to_f8, _type,
                      group_by_expert)


class GatedExperts:
    """y[t] = down[e] @ (act(gate[e] @ x[t]) * (up[e] @ x[t])), e the expert of t, zeros for a token of no expert, as in Experts.
    gate_up: [experts, 2 features, features in], an expert's gate before its up; down: [experts, features out, features]; one of
    FP32, FP16 and BF16 on the GPU.  activation: SILU, GELU, GELU_TANH or RELU; mode, gradient_mode: as in Experts.  The layer keeps
    the matrices themselves, but a copy of those that are not contiguous."""

    def __init__(self, handle, gate_up, down, activation=lib.SILU, mode=lib.FP16TCEC, gradient_mode=lib.TF32TCEC):
        _type(gate_up)
        count, twice, inner = _sizes("gate_up", gate_up)
        _, out, features = _sizes("down", down)
        if twice % 2 != 0:
            raise ValueError(f"gate_up has {twice} features, not two matrices of the same number")
        _expect("down", down, (count, out, twice // 2), gate_up.device, gate_up.dtype)
        if activation not in (lib.SILU, lib.GELU, lib.GELU_TANH, lib.RELU):
            raise ValueError(f"activation {activation}")
        self.handle, self.gate_up, self.down = handle, gate_up.contiguous(), down.contiguous()
        self.activation, self.mode, self.gradient_mode = activation, mode, gradient_mode

    def forward(self, x, experts):
        """(y, what backward needs); x and y are of the matrices' type"""
        import torch
        w, down = self.gate_up, self.down
        count, out, f = down.shape
        inner = w.shape[2]
        _expect("x", x, (len(x), inner), w.device, w.dtype)
        _expect("experts", experts, (len(x),), w.device)
        order, offsets = group_by_expert(experts, count)
        grouped, n, type = x[order], len(x), _type(x)
        h = torch.empty(n, f, device=x.device, dtype=x.dtype)
        z = torch.empty(n, 2 * f, device=x.device, dtype=x.dtype)
        y = torch.zeros(n, out, device=x.device, dtype=x.dtype)  # (the library writes the rows of experts' tokens only)
        with _on_current_stream(self.handle, w):
            _check(self.handle.gemm_gated(lib.OP_T, self.activation, f, n, inner, w, w[:, f:], inner, 2 * f * inner, grouped, inner, h, f,
                                          z, z[:, f:], 2 * f, offsets, count, self.mode, type))
            _check(self.handle.gemm_grouped(lib.OP_T, out, n, f, 1.0, down, f, out * f, h, f, 0.0, y, out, offsets, count, self.mode,
                                            type, type))
        return torch.empty_like(y).index_copy_(0, order, y), (grouped, z, order, offsets)

    def backward(self, saved, dy, d_gate_up=None, d_down=None):
        """(gradient of x, of gate_up, of down), those of matrices in FP32: added to d_gate_up and d_down, FP32 and contiguous, if
        there are such"""
        import torch
        grouped, z, order, offsets = saved
        w, down = self.gate_up, self.down
        count, out, f = down.shape
        n, inner = len(order), w.shape[2]
        _expect("x of what forward saved", grouped, (n, inner), w.device, w.dtype)
        _expect("projections of what forward saved", z, (n, 2 * f), w.device, w.dtype)
        _expect("order of what forward saved", order, (n,), w.device, torch.int64)
        _expect("offsets of what forward saved", offsets, (count + 1,), w.device, torch.int32)
        _expect("dy", dy, (n, out), w.device, w.dtype)
        betas = []
        for name, d, like in (("d_gate_up", d_gate_up, w), ("d_down", d_down, down)):
            if d is not None:
                _expect(name, d, like.shape, w.device, torch.float32)
                if not d.is_contiguous():
                    raise ValueError(f"{name} is not contiguous")
            betas.append(0.0 if d is None else 1.0)
        if d_gate_up is None:
            d_gate_up = torch.empty(w.shape, device=w.device, dtype=torch.float32)
        if d_down is None:
            d_down = torch.empty(down.shape, device=w.device, dtype=torch.float32)
        dy, type, mode = dy[order], _type(dy), self.gradient_mode
        h = torch.empty(n, f, device=w.device, dtype=w.dtype)
        dz = torch.empty_like(z)
        dx = torch.zeros_like(grouped)
        with _on_current_stream(self.handle, w):
            _check(self.handle.gemm_gated_backward(lib.OP_N, self.activation, f, n, out, down, f, out * f, dy, out, z, z[:, f:], 2 * f, dz,
                                                   dz[:, f:], 2 * f, h, f, offsets, count, mode, type))
            _check(self.handle.gemm_grouped(lib.OP_N, inner, n, 2 * f, 1.0, w, inner, 2 * f * inner, dz, 2 * f, 0.0, dx, inner, offsets,
                                            count, mode, type, type))
            # (stored as the matrices are: rows of what went in times rows of what came back)
            _check(self.handle.gemm_grouped_k(inner, 2 * f, n, 1.0, grouped, inner, dz, 2 * f, betas[0], d_gate_up, inner, 2 * f * inner,
                                              offsets, count, mode, type, lib.R_32F))
            _check(self.handle.gemm_grouped_k(f, out, n, 1.0, h, f, dy, out, betas[1], d_down, f, out * f, offsets, count, mode, type,
                                              lib.R_32F))
        return torch.empty_like(dx).index_copy_(0, order, dx), d_gate_up, d_down

    def to_f8(self):
        """The same block for serving, in 8-bit floating point (E4M3) with a scale for 128 x 128 of each matrix."""
        count, out, f = self.down.shape
        inner = self.gate_up.shape[2]
        # (blocks of an expert's two matrices: none has rows of both)
        q, scale = _matrices_to_f8(self.handle, self.gate_up.view(2 * count, f, inner))
        return F8GatedExperts(self.handle, q.view(count, 2 * f, inner), scale.view(count, 2, _blocks(f), _blocks(inner)),
                              *_matrices_to_f8(self.handle, self.down), activation=self.activation)


class F8GatedExperts:
    """GatedExperts in E4M3: gate_up with scales [experts, 2, ceil(features / 128), ceil(in / 128)], down with scales [experts,
    ceil(out / 128), ceil(features / 128)]."""

    def __init__(self, handle, gate_up, gate_up_scale, down, down_scale, activation=lib.SILU):
        import torch
        count, twice, inner = _sizes("gate_up", gate_up)
        if twice % 2 != 0:
            raise ValueError(f"gate_up has {twice} features, not two matrices of the same number")
        f = twice // 2
        _expect("gate_up", gate_up, (count, twice, inner), gate_up.device, torch.float8_e4m3fn)
        _expect("scale of gate_up", gate_up_scale, (count, 2, _blocks(f), _blocks(inner)), gate_up.device, torch.float32)
        _expect("down", down, (count, _sizes("down", down)[1], f), gate_up.device)
        if activation not in (lib.SILU, lib.GELU, lib.GELU_TANH, lib.RELU):
            raise ValueError(f"activation {activation}")
        self.handle, self.activation = handle, activation
        self.gate_up, self.gate_up_scale = gate_up.contiguous(), gate_up_scale.contiguous()
        self.down, self.down_scale = _f8_matrices("down", down, down_scale)

    def forward(self, x, experts):
        """x in FP32, FP16 or BF16, a scale taken for each 128 values of a token, and of the block's own; y of the same type"""
        import torch
        type = _type(x)
        w, down = self.gate_up, self.down
        count, out, f = down.shape
        inner, n = w.shape[2], len(x)
        _expect("x", x, (n, inner), w.device)
        _expect("experts", experts, (n,), x.device)
        order, offsets = group_by_expert(experts, count)
        grouped = x[order]
        # (zeros: rows of no expert are not written, but quantised)
        h = torch.zeros(n, f, device=x.device, dtype=x.dtype)
        y = torch.zeros(n, out, device=x.device, dtype=x.dtype)
        per = _blocks(f) * _blocks(inner)
        with _on_current_stream(self.handle, w):
            q, scale = _tokens_to_f8(self.handle, grouped)
            _check(self.handle.gemm_gated_f8(self.activation, f, n, inner, w, w[:, f:], inner, 2 * f * inner, lib.R_8F_E4M3,
                                             self.gate_up_scale, self.gate_up_scale[:, 1:], 2 * per, q, inner, lib.R_8F_E4M3, scale, h,
                                             f, type, offsets, count))
            q, scale = _tokens_to_f8(self.handle, h)
            _check(self.handle.gemm_f8(lib.OP_T, out, n, f, down, f, out * f, lib.R_8F_E4M3, self.down_scale, _blocks(out) * _blocks(f), q,
                                       f, lib.R_8F_E4M3, scale, y, out, type, offsets, count))
        return torch.empty_like(y).index_copy_(0, order, y)


def gated_reference(gate_up, down, x, experts, dy, activation=lib.SILU):
    """y, dx, d_gate_up and d_down in FP64, expert by expert, gradients by torch."""
    import torch
    act = {lib.SILU: torch.nn.functional.silu, lib.GELU: torch.nn.functional.gelu, lib.RELU: torch.nn.functional.relu,
           lib.GELU_TANH: lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[activation]
    w, v = gate_up.double().requires_grad_(), down.double().requires_grad_()
    x, dy = x.double().requires_grad_(), dy.double()
    f = down.shape[2]
    y = torch.zeros_like(dy)
    for e in range(len(w)):
        rows = torch.nonzero(experts == e)[:, 0]
        h = act(x[rows] @ w[e, :f].t()) * (x[rows] @ w[e, f:].t())
        y = y.index_copy(0, rows, h @ v[e].t())
    return (y.detach(), *torch.autograd.grad(y, (x, w, v), dy))


def main(argv=None):
    """Prints one line for each result; returns {result: relative error against FP64}."""
    import torch
    args = [int(a) for a in (sys.argv[1:] if argv is None else argv)]
    tokens, inner, features, count = args + [1000, 512, 768, 8][len(args):]
    g = torch.Generator(device="cuda").manual_seed(1)
    gate_up = torch.randn(count, 2 * features, inner, generator=g, device="cuda") * inner ** -0.5
    down = torch.randn(count, inner, features, generator=g, device="cuda") * features ** -0.5
    x = torch.randn(tokens, inner, generator=g, device="cuda")
    dy = torch.randn(tokens, inner, generator=g, device="cuda")
    experts = torch.randint(count, (tokens,), generator=g, device="cuda")
    handle = lib.Handle(stream=torch.cuda.current_stream())
    errors = {}

    def report(name, got, want):
        errors[name] = float((got.double() - want).norm() / want.norm())
        print(f"{name:24s} relative error {errors[name]:.2e}")

    for name, dtype in (("FP32", torch.float32), ("BF16", torch.bfloat16)):
        layer = GatedExperts(handle, gate_up.to(dtype), down.to(dtype))
        xs, ds = x.to(dtype), dy.to(dtype)
        y, saved = layer.forward(xs, experts)
        want = gated_reference(layer.gate_up, layer.down, xs, experts, ds)
        for part, got, exact in zip(("y", "dx", "d_gate_up", "d_down"), (y, *layer.backward(saved, ds)), want):
            report(f"{name} {part}", got, exact)
    report("8-bit floats y", GatedExperts(handle, gate_up, down).to_f8().forward(x, experts), gated_reference(gate_up, down, x, experts, dy)[0])
    torch.cuda.synchronize()
    handle.close()
    return errors


if __name__ == "__main__":
    main()
