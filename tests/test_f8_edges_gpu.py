"""Feed-forward operators in 8-bit floating point at the edges of their ranges: streams, masks and values as large or as small as their types allow."""
import pytest

from test_f8_gpu import _codes, _rand, _scales, acc  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- streams -----------------------------------------------------------------------------------------------------------

def test_a_call_on_another_stream_takes_no_memory_with_work_pending_on_this_one(acc):  # noqa: F811
    """Blocks freed a moment ago on the current stream, whose kernels have yet to write them, and calls on a stream that waits for none of that: results, plans and
    scratch memory are what they are without it."""
    import torch
    tokens, experts, k, hidden, inner = 24, 16, 4, 256, 256
    w13, s13 = _codes(3, experts, 2, inner, hidden).cuda(), (0.01 * _scales(5, experts, 2, 2, 2)).cuda()
    w2, s2 = _codes(4, experts, hidden, inner).cuda(), (0.02 * _scales(6, experts, 2, 2)).cuda()
    a, sa, b, sb = _codes(7, 200, 9000).cuda(), _scales(8, 200, 71).cuda(), _codes(9, 130, 9000).cuda(), _scales(10, 2, 71).cuda()  # (K in slices)

    def path(i, stream=None):
        x, logits = inputs[i]
        ids, weights = acc.route_experts(logits, k, stream=stream)
        plan = acc.plan_experts(ids, experts, stream=stream)
        q, s = acc.quantize_f8(x, stream=stream)
        grad = acc.route_experts_backward(logits, ids, weights, stream=stream)
        y = acc.expert_ffn_f8(x, ids, weights, w13, s13, w2, s2, stream=stream)
        c = acc.gemm_f8(a, sa if i else 2 * sa, b.t(), sb.t(), out[i], stream=stream)
        z = acc.combine_experts(rows[i], plan, weights, stream=stream)
        return ids, weights, plan._all[:2 * tokens * k + experts + 1], q, s, grad, y, c, z
    inputs = [(_rand(i, tokens, hidden).to(torch.bfloat16).cuda(), _rand(20 + i, tokens, experts).cuda()) for i in range(2)]
    rows = [_rand(30 + i, tokens * k, 100).cuda() for i in range(2)]
    out = [torch.empty((200, 130), device="cuda") for _ in range(2)]
    want = [t.clone() for t in path(1)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    path(1, side.cuda_stream)
    torch.cuda.synchronize()
    for _ in range(3):
        torch.cuda._sleep(20_000_000)
        path(0)  # (behind the sleep: its results' memory is free again, its kernels have not run)
        got = path(1, side.cuda_stream)
        torch.cuda.synchronize()
        for n, (g, w) in enumerate(zip(got, want)):
            assert torch.equal(g.view(torch.uint8), w.view(torch.uint8)) if n == 3 else torch.equal(g, w), n


def test_results_of_another_stream_may_be_used_on_this_one(acc):  # noqa: F811
    """A result that the current stream reads, having waited for the other, and that is dropped then: the other stream's next result does not take its memory before it is read."""
    import torch
    x = [_rand(i, 500, 1024).cuda() for i in range(2)]
    want = [acc.quantize_f8(v)[0].float() for v in x]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        q, _ = acc.quantize_f8(x[0], stream=side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda._sleep(20_000_000)
        read = q.float()
        del q
        other, _ = acc.quantize_f8(x[1], stream=side.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(read, want[0]) and torch.equal(other.float(), want[1])


def test_streams_by_number(acc):  # noqa: F811
    """The current stream by its own number, the default one from a stream of its own, and a ctypes pointer."""
    import ctypes
    import torch
    x = _rand(1, 40, 300).cuda()
    want = acc.quantize_f8(x)[0].float()
    torch.cuda.synchronize()
    assert torch.equal(acc.quantize_f8(x, stream=torch.cuda.current_stream().cuda_stream)[0].float(), want)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q = acc.quantize_f8(x, stream=0)[0]
        side.wait_stream(torch.cuda.default_stream())
        assert torch.equal(q.float(), want)
        q = acc.quantize_f8(x, stream=ctypes.c_void_p(0))[0]
        side.wait_stream(torch.cuda.default_stream())
        assert torch.equal(q.float(), want)
        assert torch.cuda.current_stream() == side
