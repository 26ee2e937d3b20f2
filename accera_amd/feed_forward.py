"""Feed-forward layers from the operators of f8.py, as a model uses them: a routed layer for serving, and the differentiable pieces of a dense
layer and of a router for training.

    layer = ExpertLayer(router, gate, up, down, top_k=6)       # 16-bit or fp32 weights, quantised once
    y = layer(x)                                               # router, choice of experts, their products, weighted sum

    y = f8_linear(x, w)                                        # y = x @ w.T; both gradients are block-scaled products too
    ids, weights = f8_route(logits, top_k)                     # weights carry a gradient to the logits

Run as a command it times a decoding step, a prompt batch and a training step of random weights, and says how far each is from the same layer in
fp32:

    python -m accera_amd.feed_forward [--tokens 8 1024] [--hidden 2048] [--inner 1024] [--experts 64] [--top-k 6] [--type bf16]
"""
import argparse

import torch

from . import _lib
from .f8 import BLOCK, F8, expert_ffn_f8, gemm_f8, quantize_f8, route_experts, route_experts_backward, without_gradient
from .gemm import gemm_relu


class ExpertLayer:
    """A routed feed-forward layer with weights in e4m3: out[t] = sum over t's experts of weight * down(silu(gate(x[t])) * up(x[t])).

    router (hidden, experts) fp16 / bf16; gate, up (experts, inner, hidden) and down (experts, hidden, inner) fp32 / fp16 / bf16, quantised here in blocks
    of 128 x 128.  ``route``: further arguments of route_experts.  For serving: it has no gradient, and says so where one is asked for.
    """

    def __init__(self, router, gate, up, down, top_k, **route):
        experts, inner, hidden = gate.shape
        if up.shape != gate.shape or down.shape != (experts, hidden, inner) or router.shape != (hidden, experts):
            raise ValueError(f"shape mismatch: router {tuple(router.shape)}, gate {tuple(gate.shape)}, up {tuple(up.shape)}, down {tuple(down.shape)}")
        hidden_blocks, inner_blocks = -(-hidden // BLOCK), -(-inner // BLOCK)
        self.router, self.top_k, self.route = router, top_k, route
        self.w13 = gate.new_empty((experts, 2, inner, hidden), dtype=F8)
        self.w13_scale = gate.new_empty((experts, 2, inner_blocks, hidden_blocks), dtype=torch.float32)
        self.w2 = gate.new_empty((experts, hidden, inner), dtype=F8)
        self.w2_scale = gate.new_empty((experts, hidden_blocks, inner_blocks), dtype=torch.float32)
        for e in range(experts):
            quantize_f8(gate[e], self.w13[e, 0], self.w13_scale[e, 0], group_rows=BLOCK)
            quantize_f8(up[e], self.w13[e, 1], self.w13_scale[e, 1], group_rows=BLOCK)
            quantize_f8(down[e], self.w2[e], self.w2_scale[e], group_rows=BLOCK)

    def choose(self, x):
        """(ids, weights) of the experts of x (tokens, hidden), in the router's type; fp32 scores."""
        logits = x.new_empty((x.shape[0], self.router.shape[1]), dtype=torch.float32)
        gemm_relu(x, self.router, logits, epilogue=_lib.EPILOGUE_NONE)
        ids, weights = route_experts(logits, self.top_k, **self.route)
        return ids, without_gradient("ExpertLayer", weights, x, self.router)

    def __call__(self, x, out=None):
        with torch.no_grad():
            ids, weights = self.choose(x)
            y = expert_ffn_f8(x, ids, weights, self.w13, self.w13_scale, self.w2, self.w2_scale, out=out)
        return without_gradient("ExpertLayer", y, x, self.router)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        xq, xs = quantize_f8(x)
        wq, ws = quantize_f8(w, group_rows=BLOCK)
        return gemm_f8(xq, xs, wq.t(), ws.t(), x.new_empty((x.shape[0], w.shape[0])))

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dyq, dys = quantize_f8(dy)
            wq, ws = quantize_f8(w, group_rows=BLOCK, transpose=True)
            dx = gemm_f8(dyq, dys, wq.t(), ws.t(), torch.empty_like(x, memory_format=torch.contiguous_format))
            dx = without_gradient("the gradient of f8_linear", dx, dy, x, w)  # (in a backward pass that is to be differentiated itself)
        if ctx.needs_input_grad[1]:
            # (groups run along the tokens that are summed over; the sum over a batch stays in fp32 until it is the weight's type)
            dyq, dys = quantize_f8(dy, transpose=True)
            xq, xs = quantize_f8(x, transpose=True)
            dw = gemm_f8(dyq, dys, xq.t(), xs.t(), w.new_empty(w.shape, dtype=torch.float32)).to(w.dtype)
            dw = without_gradient("the gradient of f8_linear", dw, dy, x, w)
        return dx, dw


def f8_linear(x, w):
    """x (tokens, in) @ w (out, in).T in x's type, operands of this product and of both gradients' in e4m3 (once: the gradients have none of their own)."""
    return _Linear.apply(x, w)


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, options):
        ids, weights = route_experts(logits, top_k, **options)
        ctx.save_for_backward(logits, ids)
        ctx.options = {name: options[name] for name in ("score", "renormalise", "scale") if name in options}
        ctx.mark_non_differentiable(ids)
        return ids, weights

    @staticmethod
    def backward(ctx, _, dweights):
        logits, ids = ctx.saved_tensors
        grad = route_experts_backward(logits, ids, dweights.contiguous(), **ctx.options)
        return without_gradient("the gradient of f8_route", grad, logits, dweights), None, None


def f8_route(logits, top_k, **options):
    """route_experts with a gradient: of the weights, through the scores, to the logits (the choice itself has none)."""
    return _Route.apply(logits, top_k, options)


def _expert_layer_fp32(x, router, gate, up, down, top_k):
    logits = x.float() @ router.float()
    scores, ids = torch.topk(torch.softmax(logits, dim=1), top_k, dim=1)
    scores = scores / scores.sum(dim=1, keepdim=True)
    y = torch.zeros(x.shape, device=x.device)
    for e in range(gate.shape[0]):
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        v = x[token].float()
        h = torch.nn.functional.silu(v @ gate[e].float().t()) * (v @ up[e].float().t())
        y.index_add_(0, token, scores[token, slot, None] * (h @ down[e].float().t()))
    return y


def _microseconds(run, times=20):
    for _ in range(3):
        run()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(times):
        run()
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) * 1e3 / times


def _apart(a, b):
    a, b = a.detach().float(), b.detach().float()
    return float((a - b).norm() / b.norm())


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--tokens", type=int, nargs="+", default=[8, 1024])
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--inner", type=int, default=1024)
    ap.add_argument("--experts", type=int, default=64)
    ap.add_argument("--top-k", type=int, default=6)
    ap.add_argument("--type", choices=("bf16", "fp16"), default="bf16")
    a = ap.parse_args(argv)
    dtype = torch.bfloat16 if a.type == "bf16" else torch.float16
    gen = torch.Generator(device="cuda").manual_seed(0)

    def rand(*shape, scale=1.0):
        return (scale * torch.randn(shape, generator=gen, device="cuda")).to(dtype)

    router = rand(a.hidden, a.experts, scale=a.hidden ** -0.5)
    gate, up = (rand(a.experts, a.inner, a.hidden, scale=a.hidden ** -0.5) for _ in range(2))
    down = rand(a.experts, a.hidden, a.inner, scale=a.inner ** -0.5)
    layer = ExpertLayer(router, gate, up, down, a.top_k)
    for tokens in a.tokens:
        x = rand(tokens, a.hidden)
        print(f"routed layer, {tokens} tokens: {_microseconds(lambda: layer(x)):.1f} us, {_apart(layer(x), _expert_layer_fp32(x, router, gate, up, down, a.top_k)):.3f} from fp32",
              flush=True)
    tokens = max(a.tokens)
    x, w, dy = rand(tokens, a.hidden).requires_grad_(), gate[0].clone().requires_grad_(), rand(tokens, a.inner)

    def step():
        x.grad = w.grad = None
        f8_linear(x, w).backward(dy)
    t = _microseconds(step)
    far = (_apart(f8_linear(x, w), x.float() @ w.float().t()), _apart(x.grad, dy.float() @ w.float()), _apart(w.grad, dy.float().t() @ x.float()))
    print(f"dense layer {a.inner} x {a.hidden}, forward and backward, {tokens} tokens: {t:.1f} us, output {far[0]:.3f}, gradients {far[1]:.3f} and {far[2]:.3f} from fp32")


if __name__ == "__main__":
    main()
