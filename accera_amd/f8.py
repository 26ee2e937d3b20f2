"""Device-tensor front end of the feed-forward operators in 8-bit floating point (include/accera_mi355x_f8.h): quantising to
e4m3, the block-scaled product, routing to experts and the experts' products.  torch supplies device memory and streams, every
computation happens in the HIP kernels of libaccera_mi355x.so.

Calls are asynchronous on the current stream of the tensors' device, or on ``stream`` (a raw hipStream_t), which then has to wait by itself for whatever
makes the inputs.  Results that are not passed in are allocated, as torch's allocator does it for work on that stream; under a graph capture that works as for
any torch allocation.

None of them has a gradient by itself (feed_forward.f8_linear and f8_route do).  Where an input of a routed layer, a weighted sum or a choice asks for one, the
result carries a node that refuses it.

A layer y = x @ W.T, with W (N, K):

    wq, ws = quantize_f8(W, group_rows=128)                 # once
    xq, xs = quantize_f8(x)
    gemm_f8(xq, xs, wq.t(), ws.t(), y)

and its gradients:

    dyq, dys = quantize_f8(dy)
    wtq, wts = quantize_f8(W, group_rows=128, transpose=True)
    gemm_f8(dyq, dys, wtq.t(), wts.t(), dx)                 # dx = dy @ W
    dytq, dyts = quantize_f8(dy, transpose=True)
    xtq, xts = quantize_f8(x, transpose=True)
    gemm_f8(dytq, dyts, xtq.t(), xts.t(), dw)               # dw = dy.T @ x
"""
import ctypes
import importlib.machinery
import importlib.util
import os

import torch

from . import _lib

F8 = torch.float8_e4m3fn
BLOCK = 128

_ACTIVATIONS = {"none": 0, "relu": 1, "silu_mul": 2}
_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"best": 0, "best_two": 1}


def _load():
    """csrc/torch_f8.cpp: what checks the tensors of a call, allocates its results and calls the library."""
    _lib.lib()
    path = os.path.join(os.path.dirname(_lib.LIB_PATH), "_torch_f8.so")
    if not os.path.exists(path):
        raise RuntimeError(f"{path} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` (or `make -C accera_amd/csrc`).")
    loader = importlib.machinery.ExtensionFileLoader("_torch_f8", path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_torch_f8", loader))
    loader.exec_module(module)
    return module


_native = _load()


def _raw(stream):
    return (stream.value or 0) if isinstance(stream, ctypes.c_void_p) else stream


class _Refused(torch.autograd.Function):
    """A result as it is, whose gradient is an error: without this, autograd would take what made it for a constant."""

    @staticmethod
    def forward(ctx, name, y, *inputs):
        ctx.name = name
        return y.view_as(y)

    @staticmethod
    def backward(ctx, dy):
        raise RuntimeError(f"{ctx.name} has no gradient: call it under torch.no_grad(), or with inputs that are detached")


def without_gradient(name, y, *inputs):
    """y, the result of ``name`` for these inputs, with a gradient that is refused if any of them asks for one."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs):
        return _Refused.apply(name, y, *inputs)
    return y


def quantize_f8(x, out=None, scale=None, *, group_rows=1, transpose=False, activation="none", power_of_two=False, stream=None):
    """(q, scale): e4m3 values and fp32 block scales of act(x), a matrix of fp32 / fp16 / bf16; q * scale (spread over its blocks) is
    what they stand for.

    Groups of 128 run along q's last axis; ``group_rows`` (1, or 128 for a weight) rows share a scale.  ``transpose``: q is the
    transposed matrix.  ``activation``: "none", "relu", or "silu_mul" of x = [gate | up] (q is half as wide).  ``power_of_two``:
    scales are powers of two, so that only the codes are rounded.  An all-zero group has the scale 2^-126; an infinity or NaN makes its whole
    group NaN, behind a ReLU too (a product's ReLU makes NaN 0).

    q (rows, cols) has rows that start on 16-byte boundaries unless ``out`` says otherwise; scale is (ceil(rows / group_rows), ceil(cols / 128)),
    laid out by blocks for single rows, as the product reads them.
    """
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}")
    return _native.quantize(x, out, scale, group_rows, transpose, act, power_of_two, _raw(stream))


def gemm_f8(A, a_scale, B, b_scale, C, epilogue=_lib.EPILOGUE_NONE, variant=_lib.VARIANT_AUTO, k_slices=0, stream=None):
    """C = epilogue(A @ B) of e4m3 operands with block scales, in place on C (fp32 / fp16 / bf16), asynchronously.

    A (M, K) with a_scale (M, ceil(K / 128)); B (K, N) with b_scale (ceil(K / 128), ceil(N / 128)), or (ceil(K / 128), N) for scales of single columns
    (as many columns as rows of b_scale are told apart by N; where both are the same, N = 1, they are the same thing).  ``epilogue``: NONE
    or RELU.  B is commonly ``wq.t()`` of a weight quantised by rows, b_scale ``ws.t()``.  Strides are honoured; operands that are
    contiguous along K, with rows on 16-byte boundaries (as quantize_f8 leaves them), are taken as they lie, others laid out anew first.  A small result with a long sum is computed in slices
    of K, added in a fixed order; ``variant`` and ``k_slices`` name a kernel and a number of slices (of a tile kernel) instead.

    A fp32 C has fp32 sums.  fp16 and bf16 ones are computed twice as fast on the e4m3 matrix instruction, whose sums inside a block of 128 drop what lies below 2^-13 of the
    largest of eight terms: 2^-16 of the result, more where terms cancel.  Where that matters take a fp32 C, or name a variant with fp32 sums (0, 6 to 8, 18, 19).
    """
    _native.gemm(A, a_scale, B, b_scale, C, epilogue, variant, k_slices, _raw(stream))
    return C


def route_experts(logits, top_k, *, score="softmax", bias=None, groups=1, top_groups=None, group_score=None, renormalise=True, scale=1.0, stream=None):
    """(ids, weights) of the experts each token goes to: (tokens, top_k) int32, best first, and fp32.

    The score is the ``softmax`` over the experts or the ``sigmoid`` of the logits (tokens, experts); ``bias`` (fp32 per expert) is added to it for
    the choice only.  With ``groups`` > 1 only the experts of the ``top_groups`` best groups (of neighbouring experts) are chosen
    from; a group's score is that of its "best" expert or the sum of its "best_two" (the default for softmax / sigmoid).  Ties go to the
    lowest expert.  weights = scale * score, divided by the sum over the token's experts if ``renormalise``.  An expert whose logit
    or bias is -inf is never chosen; slots that are left have id -1 and weight 0.
    """
    code = _SCORES.get(score)
    if code is None:
        raise ValueError(f"unknown score {score!r}")
    of_group = code if group_score is None else _GROUP_SCORES.get(group_score)
    if of_group is None:
        raise ValueError(f"unknown group_score {group_score!r}")
    ids, weights = _native.route(logits, top_k, code, bias, groups, top_groups, of_group, renormalise, scale, _raw(stream))
    return ids, without_gradient("route_experts", weights, logits) if logits.requires_grad else weights


def route_experts_backward(logits, ids, dweights, *, score="softmax", renormalise=True, scale=1.0, out=None, stream=None):
    """Gradient of ``logits`` (its type) from the gradient ``dweights`` of the weights that route_experts gave with these ids and arguments."""
    code = _SCORES.get(score)
    if code is None:
        raise ValueError(f"unknown score {score!r}")
    return _native.route_backward(logits, ids, dweights, code, renormalise, scale, out, _raw(stream))


class ExpertPlan:
    """The (token, slot) pairs in the order of their experts: order[r] is the pair token * top_k + slot of sorted row r, position[token, slot]
    its row (-1: the pair has no expert), offsets[e] the first row of expert e (experts + 1 of them).  int32 on the GPU."""

    __slots__ = ("tokens", "top_k", "experts", "_all")

    def __init__(self, tokens, top_k, experts, all_):
        self.tokens, self.top_k, self.experts = tokens, top_k, experts
        self._all = all_  # order, position, offsets (and scratch memory) in one tensor; the views are made when they are asked for

    order = property(lambda self: self._all[:self.tokens * self.top_k])
    position = property(lambda self: self._all[self.tokens * self.top_k:2 * self.tokens * self.top_k].view(self.tokens, self.top_k))
    offsets = property(lambda self: self._all[2 * self.tokens * self.top_k:2 * self.tokens * self.top_k + self.experts + 1])


def plan_experts(ids, experts, stream=None):
    """The ExpertPlan of ids (tokens, top_k) int32; a number outside 0 .. experts - 1 means no expert, and its pair comes last."""
    return ExpertPlan(ids.shape[0], ids.shape[-1], experts, _native.plan(ids, experts, _raw(stream)))


def expert_gemm_f8(A, a_scale, B, b_scale, plan, C, *, gather, row_weights=None, variant=_lib.VARIANT_AUTO, stream=None):
    """Row r of C = A's row for sorted row r of ``plan`` times the matrix of r's expert, in place on C (pairs, N), asynchronously.

    ``gather``: A (tokens, K) has one row per token; otherwise (pairs, K), one per sorted row.  B (experts, K, N), b_scale (experts, ceil(K / 128),
    ceil(N / 128)), commonly ``wq.transpose(1, 2)`` of (experts, N, K) weights: contiguous along K.  ``row_weights`` (tokens, top_k) fp32 multiply the
    rows of their pairs before these are rounded.  Rows of C that belong to no expert are left as they are.
    """
    _native.expert_gemm(A, a_scale, B, b_scale, plan._all, plan.tokens, plan.top_k, plan.experts, C, gather, row_weights, variant, _raw(stream))
    return C


def combine_experts(x, plan, weights=None, out=None, stream=None):
    """y[t] = sum over t's slots of weights[t, slot] * x[plan.position[t, slot]] (weights None: of 1), fp32 sums, in x's type."""
    return without_gradient("combine_experts", _native.combine(x, plan._all, plan.tokens, plan.top_k, weights, out, _raw(stream)), x, weights)


def expert_ffn_f8(x, ids, weights, w13, w13_scale, w2, w2_scale, out=None, workspace=None, stream=None):
    """A routed feed-forward layer: out[t] = sum over t's slots of weights[t, slot] * W2[e] q(silu(W1[e] q(x[t])) * (W3[e] q(x[t]))), e = ids[t, slot].

    x (tokens, hidden) fp16 / bf16; ids, weights as route_experts gives them (an id outside 0 .. experts - 1: no expert).  w13 (experts, 2, inner, hidden):
    gate and up, w2 (experts, hidden, inner), e4m3 with scales of 128 x 128 blocks, contiguous.  q quantises rows with power-of-two scales, so that the inner values
    are rounded once, to their codes.  Up to 16 rows for each expert all sums are fp32; with more, some are the e4m3 instruction's (see gemm_f8: the gate and up product's of a bf16 layer,
    the down product's), and a bf16 layer's rows are fp16 with shared powers of two until they are added up, in fp32.  ``workspace``: a uint8 tensor of
    at least expert_ffn_workspace(...) bytes to be used over and over (on one stream: calls that may run at the same time take one each), or None to allocate one.
    """
    y = _native.expert_ffn(x, ids, weights, w13, w13_scale, w2, w2_scale, out, workspace, _raw(stream))
    return without_gradient("expert_ffn_f8", y, x, weights) if x.requires_grad or weights.requires_grad else y


def expert_ffn_workspace(tokens, hidden, inner, experts, top_k):
    """Bytes of scratch memory that expert_ffn_f8 takes for these sizes (negative: it refuses them)."""
    return _lib.lib().acc950_f8_expert_ffn_workspace(tokens, hidden, inner, experts, top_k)
