"""One layer of experts on the library's grouped products: each token is multiplied with the matrix of its expert.

    python -m cumpsgemm_amd.experts [tokens [features_in [features_out [experts]]]]

runs a training step in FP32 on split operands and in BF16 (forward, the gradients of tokens and matrices), then serves
the trained matrices in 8-bit integers, and prints how far each result is from FP64.

Tensors hold a token (an output channel) in a row, which the library's column-major calls read as a column.  All work goes to
torch's current stream, whichever the handle has; it is back on its own afterwards, behind that work."""
import contextlib
import sys

from . import _lib as lib


def group_by_expert(experts, count):
    """(order, offsets): the tokens' numbers sorted by expert (those of one expert in their order), and where each expert's
    begin, `count` + 1 int32.  On the tensor's own device, without waiting for it.  Tokens of no expert (numbers below 0 or
    from `count` on) come before the first one's and behind the last one's."""
    import torch
    if not experts.dtype.is_floating_point:  # (`count` itself need not fit the type that the numbers have)
        experts = experts.to(torch.promote_types(experts.dtype, torch.int32))
    order = torch.argsort(experts, stable=True)
    first = torch.arange(count + 1, device=experts.device, dtype=experts.dtype)
    return order, torch.searchsorted(experts[order], first).to(torch.int32)


def _type(t):
    import torch
    types = {torch.float32: lib.R_32F, torch.float16: lib.R_16F, torch.bfloat16: lib.R_16BF}
    if t.dtype not in types:
        raise ValueError(f"{t.dtype}: not FP32, FP16 or BF16")
    return types[t.dtype]


def _expect(name, t, shape, device, dtype=None):
    """The library is given addresses, sizes and one type for all operands: ValueError for a tensor that is not as those say."""
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} is of {t.dtype}, not of {dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} is {list(t.shape)}, not {list(shape)}")


def _sizes(name, weights):
    """experts, features out, features in"""
    if weights.dim() != 3:
        raise ValueError(f"{name} are {list(weights.shape)}, not [experts, features out, features in]")
    return weights.shape


def _check(status):
    if status != lib.STATUS_SUCCESS:
        raise RuntimeError(f"hipblasStatus {status}")


def _stream_of(t):
    """The address of torch's current stream on the GPU that t is on."""
    import torch
    if not t.is_cuda:
        raise ValueError(f"weights on {t.device}, not on the GPU")
    return torch.cuda.current_stream(t.device).cuda_stream


@contextlib.contextmanager
def _on_current_stream(handle, weights):
    """The library's calls between torch's own, on one stream with them."""
    before = handle.stream
    handle.set_stream(_stream_of(weights))
    try:
        yield
    finally:
        if handle.stream != before:
            handle.set_stream(before)


class Experts:
    """y[t] = weights[expert of t] @ x[t], zeros for a token of no expert (one that was dropped: a number below 0 or from
    `experts` on), whose dy counts for nothing; weights: [experts, features out, features in], FP32, FP16 or BF16, on the GPU.
    mode, gradient_mode: how FP32 operands are multiplied, forward and for the gradients.  FP16TCEC splits into FP16 terms,
    which hold nothing beyond 65504 and are off by up to 2^-36 however small the value is: 1.5e-4 of one of 1e-7, such as the
    gradients of a mean over many tokens are (the terms of dy of 1e-6: 8.6e-6 of its norm; of 1e-9: 8.6e-3).  TF32TCEC's three
    BF16 terms have FP32's range.  The layer keeps the weights themselves, but a copy if they are not contiguous."""

    def __init__(self, handle, weights, mode=lib.FP16TCEC, gradient_mode=lib.TF32TCEC):
        _type(weights)
        _sizes("weights", weights)
        self.handle, self.weights, self.mode, self.gradient_mode = handle, weights.contiguous(), mode, gradient_mode

    def forward(self, x, experts):
        """(y, what backward needs); x and y are of the weights' type"""
        import torch
        w = self.weights
        count, out, inner = w.shape
        _expect("x", x, (len(x), inner), w.device, w.dtype)
        _expect("experts", experts, (len(x),), w.device)
        order, offsets = group_by_expert(experts, count)
        grouped = x[order]
        y = torch.zeros(len(x), out, device=x.device, dtype=x.dtype)  # (the library writes the rows of experts' tokens only)
        with _on_current_stream(self.handle, w):
            _check(self.handle.gemm_grouped(lib.OP_T, out, len(x), inner, 1.0, w, inner, out * inner, grouped, inner, 0.0, y, out,
                                            offsets, count, self.mode, _type(x), _type(y)))
        return torch.empty_like(y).index_copy_(0, order, y), (grouped, order, offsets)

    def backward(self, saved, dy, dw=None):
        """(gradient of x, gradient of the weights in FP32: added to dw, FP32 and contiguous, if there is one)"""
        import torch
        grouped, order, offsets = saved
        w = self.weights
        count, out, inner = w.shape
        _expect("x of what forward saved", grouped, (len(order), inner), w.device, w.dtype)
        _expect("order of what forward saved", order, (len(order),), w.device, torch.int64)
        _expect("offsets of what forward saved", offsets, (count + 1,), w.device, torch.int32)
        _expect("dy", dy, (len(order), out), w.device, w.dtype)
        if dw is not None:
            _expect("dw", dw, w.shape, w.device, torch.float32)
            if not dw.is_contiguous():
                raise ValueError("dw is not contiguous")
        dy = dy[order]
        dx = torch.zeros_like(grouped)
        beta = 0.0 if dw is None else 1.0
        if dw is None:
            dw = torch.empty(w.shape, device=w.device, dtype=torch.float32)
        with _on_current_stream(self.handle, w):
            _check(self.handle.gemm_grouped(lib.OP_N, inner, len(dy), out, 1.0, w, inner, out * inner, dy, out, 0.0, dx, inner,
                                            offsets, count, self.gradient_mode, _type(dy), _type(dx)))
            # (stored as the weights are, features in contiguous: rows of x times rows of dy)
            _check(self.handle.gemm_grouped_k(inner, out, len(dy), 1.0, grouped, inner, dy, out, beta, dw, inner, out * inner,
                                              offsets, count, self.gradient_mode, _type(dy), lib.R_32F))
        return torch.empty_like(dx).index_copy_(0, order, dx), dw

    def to_int8(self):
        """The same layer for serving, in 8-bit integers with a scale for each output channel."""
        import torch
        count, out, inner = self.weights.shape
        q = torch.empty(count, out, inner, device=self.weights.device, dtype=torch.int8)
        scale = torch.empty(count, out, device=self.weights.device, dtype=torch.float32)
        with _on_current_stream(self.handle, self.weights):
            _check(self.handle.quantize_i8(inner, count * out, self.weights, inner, _type(self.weights), q, inner, scale))
        return Int8Experts(self.handle, q, scale)


class Int8Experts:
    """weights: [experts, features out, features in] 8-bit integers, scale: [experts, features out].  Tokens of no expert as in
    Experts."""

    def __init__(self, handle, weights, scale):
        import torch
        count, out, inner = _sizes("weights", weights)
        _expect("weights", weights, (count, out, inner), weights.device, torch.int8)
        _expect("scale", scale, (count, out), weights.device, torch.float32)
        self.handle, self.weights, self.scale = handle, weights.contiguous(), scale.contiguous()

    def forward(self, x, experts):
        """x in FP32, FP16 or BF16, a scale taken for each token; y of the same type"""
        import torch
        _type(x)
        count, out, inner = self.weights.shape
        _expect("x", x, (len(x), inner), self.weights.device)
        _expect("experts", experts, (len(x),), x.device)
        order, offsets = group_by_expert(experts, count)
        grouped = x[order]
        q = torch.empty(len(x), inner, device=x.device, dtype=torch.int8)
        scale = torch.empty(len(x), device=x.device, dtype=torch.float32)
        y = torch.zeros(len(x), out, device=x.device, dtype=x.dtype)  # (the library writes the rows of experts' tokens only)
        with _on_current_stream(self.handle, self.weights):
            _check(self.handle.quantize_i8(inner, len(x), grouped, inner, _type(x), q, inner, scale))
            _check(self.handle.gemm_i8(out, len(x), inner, self.weights, inner, out * inner, self.scale, q, inner, scale, y, out,
                                       _type(y), offsets, count))
        return torch.empty_like(y).index_copy_(0, order, y)


def reference(weights, x, experts, dy):
    """y, dx and dw in FP64, expert by expert."""
    import torch
    w, x, dy = weights.double(), x.double(), dy.double()
    y, dx, dw = torch.empty_like(dy), torch.empty_like(x), torch.zeros_like(w)
    for e in range(len(w)):
        rows = torch.nonzero(experts == e)[:, 0]
        y[rows] = x[rows] @ w[e].t().contiguous()
        dx[rows] = dy[rows] @ w[e]
        dw[e] = dy[rows].t().contiguous() @ x[rows]
    return y, dx, dw


def main(argv=None):
    """Prints one line for each result; returns {result: relative error against FP64}."""
    import torch
    args = [int(a) for a in (sys.argv[1:] if argv is None else argv)]
    tokens, inner, out, count = args + [1000, 512, 768, 8][len(args):]
    g = torch.Generator(device="cuda").manual_seed(1)
    weights = torch.randn(count, out, inner, generator=g, device="cuda") * inner ** -0.5
    x = torch.randn(tokens, inner, generator=g, device="cuda")
    dy = torch.randn(tokens, out, generator=g, device="cuda")
    experts = torch.randint(count, (tokens,), generator=g, device="cuda")
    handle = lib.Handle(stream=torch.cuda.current_stream())
    errors = {}

    def report(name, got, want):
        errors[name] = float((got.double() - want).norm() / want.norm())
        print(f"{name:24s} relative error {errors[name]:.2e}")

    for name, dtype in (("FP32", torch.float32), ("BF16", torch.bfloat16)):
        layer = Experts(handle, weights.to(dtype))
        xs, ds = x.to(dtype), dy.to(dtype)
        y, saved = layer.forward(xs, experts)
        dx, dw = layer.backward(saved, ds)
        for part, got, want in zip(("y", "dx", "dw"), (y, dx, dw), reference(layer.weights, xs, experts, ds)):
            report(f"{name} {part}", got, want)
    report("8-bit integers y", Experts(handle, weights).to_int8().forward(x, experts), reference(weights, x, experts, dy)[0])
    torch.cuda.synchronize()
    handle.close()
    return errors


if __name__ == "__main__":
    main()
