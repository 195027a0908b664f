"""Document attention (kernels/attention_cuda.py) against 64-bit values with derived bounds."""

import random
import threading

import pytest
import torch

from attention_reference import compare, reference
from causal_tuner_b200 import _lib
from causal_tuner_b200.kernels.attention_cuda import (attention_backward, attention_forward, document_attention,
                                                      prepare_documents)

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_guard")]

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def documents(rows, width, seed, longest, gap=0, shortest=1):
    rng, spans = random.Random(seed), []
    for row in range(rows):
        start = rng.randint(0, gap)
        while start < width:
            end = min(width, start + rng.randint(shortest, longest))
            spans.append((row, start, end))
            start = end + rng.randint(0, gap)
    return tuple(spans)


def tensors(rows, width, heads, kv_heads, dim, dtype, seed=0, factor=1.0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda h: (torch.randn(rows, width, h, dim, generator=generator, device="cuda") * factor).to(TYPES[dtype])
    return make(heads), make(kv_heads), make(kv_heads), make(heads)


def covered(rows, width, spans):
    mask = torch.zeros(rows, width, dtype=torch.bool, device="cuda")
    for row, start, end in spans:
        mask[row, start:end] = True
    return mask


def run(q, k, v, dy, spans, scale=None):
    plan = prepare_documents(q.shape[:2], spans, q.device, q.shape[2], k.shape[2])
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    y = document_attention(*leaves, plan, scale=scale)
    grads = torch.autograd.grad(y, leaves, dy)
    return dict(zip(("y", "dq", "dk", "dv"), (y.detach(), *grads)))


def check(q, k, v, dy, spans, scale=None, rounded=None):
    rounded = q.dtype != torch.float32 if rounded is None else rounded
    values, errors = reference(q, k, v, spans, q.shape[-1] ** -0.5 if scale is None else scale, dy, rounded)
    actual = run(q, k, v, dy, spans, scale)
    compare(actual, values, errors)
    mask = covered(*q.shape[:2], spans)
    for name, value in actual.items():
        assert (value[~mask] == 0).all(), name
    return actual


HEADS = [(1, 1), (4, 1), (32, 1), (3, 1), (6, 2), (8, 8), (24, 8)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads, kv_heads", HEADS)
@pytest.mark.parametrize("dim", [64, 128])
def test_heads_and_types(dtype, heads, kv_heads, dim):
    spans = documents(2, 301, 7, 170)
    check(*tensors(2, 301, heads, kv_heads, dim, dtype), spans)


@pytest.mark.parametrize("dtype, dim", [("bf16", 128), ("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("heads, kv_heads", [(32, 1), (16, 16), (12, 4), (40, 8)])
@pytest.mark.parametrize("longest, gap", [(30, 0), (300, 17), (1400, 3)])
def test_more_tiles_than_the_gpu_has_sms(dtype, dim, heads, kv_heads, longest, gap):
    """Several tiles of queries, of unequal length, per persistent block; short documents leave its second stage empty."""
    spans = documents(3, 1400, 21, longest, gap=gap)
    check(*tensors(3, 1400, heads, kv_heads, dim, dtype), spans)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 385, 700])
@pytest.mark.parametrize("heads, kv_heads", [(2, 2), (4, 1)])
def test_lengths(dtype, length, heads, kv_heads):
    check(*tensors(1, length, heads, kv_heads, 64, dtype), ((0, 0, length),))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [1, 7, 8, 20, 40, 72, 80, 96, 100, 120, 127])
def test_head_dims(dtype, dim):
    check(*tensors(1, 203, 4, 2, dim, dtype), documents(1, 203, 3, 150, gap=5))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads, kv_heads", [(4, 1), (2, 2), (32, 1)])
def test_what_lies_outside_the_documents_reaches_nothing(dtype, heads, kv_heads):
    """Padding full of NaN, infinities and the types' extremes."""
    spans = documents(3, 211, 11, 90, gap=40)
    inputs = tensors(3, 211, heads, kv_heads, 64, dtype)
    mask = covered(3, 211, spans)
    for index, tensor in enumerate(inputs):
        outside = (~mask).nonzero()
        poison = (float("nan"), float("inf"), float("-inf"), torch.finfo(tensor.dtype).min)
        for i, (row, column) in enumerate(outside.tolist()):
            tensor[row, column] = poison[(i + index) % 4]
    clean = [torch.where(mask[..., None, None], t, torch.zeros_like(t)) for t in inputs]
    values, errors = reference(*clean[:3], spans, 64 ** -0.5, clean[3], dtype != "fp32")
    actual = run(*inputs, spans)
    compare(actual, values, errors)
    for value in actual.values():
        assert (value[~mask] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_a_nan_inside_a_document_stays_in_it(dtype):
    spans = ((0, 0, 100), (0, 100, 230), (0, 230, 300))
    q, k, v, dy = tensors(1, 300, 4, 1, 64, dtype)
    before = run(q, k, v, dy, spans)
    v[0, 150] = float("nan")
    k[0, 120] = float("inf")
    after = run(q, k, v, dy, spans)
    for name in before:
        for start, end in ((0, 100), (230, 300)):
            assert torch.equal(before[name][0, start:end], after[name][0, start:end]), name


def test_documents_that_follow_each_other_do_not_see_each_other():
    q, k, v, dy = tensors(1, 640, 8, 1, 128, "bf16")
    whole = run(q, k, v, dy, ((0, 0, 130), (0, 130, 131), (0, 131, 640)))
    for start, end in ((0, 130), (130, 131), (131, 640)):
        alone = run(*(t[:, start:end].contiguous() for t in (q, k, v, dy)), ((0, 0, end - start),))
        assert torch.equal(whole["y"][:, start:end], alone["y"])
        # the gradients' pieces depend on the whole batch, the values on the documents alone
        for name in ("dq", "dk", "dv"):
            a, b = whole[name][:, start:end].double(), alone[name].double()
            assert float((a - b).norm()) <= 2.0 ** -7 * float(b.norm()) + 1e-30, name


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_strided_operands(dtype):
    """q, k, v as slices of one fused projection, head-major tensors, an expanded key head, reversed dimension orders."""
    spans = documents(2, 150, 5, 140)
    generator = torch.Generator(device="cuda").manual_seed(1)
    fused = torch.randn(2, 150, 8, 64, generator=generator, device="cuda").to(TYPES[dtype])
    dy = torch.randn(2, 150, 4, 64, generator=generator, device="cuda").to(TYPES[dtype])
    q, k, v = fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:8]
    expected = run(q.contiguous(), k.contiguous(), v.contiguous(), dy, spans)
    same = lambda actual: all(torch.equal(actual[name], expected[name]) for name in expected)
    assert same(run(q, k, v, dy, spans))
    major = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    assert same(run(major(q), major(k), major(v), major(dy), spans))
    inner = lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)
    assert same(run(inner(q), inner(k), inner(v), inner(dy), spans))
    shared = k[:, :, :1]
    spread = run(q, shared.expand(2, 150, 2, 64), v, dy, spans)
    copied = run(q, shared.expand(2, 150, 2, 64).contiguous(), v, dy, spans)
    assert all(torch.equal(spread[name], copied[name]) for name in spread)
    broadcast = dy[:, :1].expand(2, 150, 4, 64)
    spread, copied = run(q, k, v, broadcast, spans), run(q, k, v, broadcast.contiguous(), spans)
    assert all(torch.equal(spread[name], copied[name]) for name in spread)


def test_operands_that_are_not_16_byte_aligned():
    spans = documents(1, 140, 2, 90)
    storage = torch.randn(140 * 4 * 64 + 1, device="cuda").to(torch.bfloat16)
    odd = storage[1:].view(1, 140, 4, 64)
    q, k, v, dy = tensors(1, 140, 4, 4, 64, "bf16")
    check(odd, k, v, dy, spans)
    check(q, odd, odd, dy, spans)
    check(q, k, v, odd, spans)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_large_scores_and_scales(dtype):
    spans = documents(1, 260, 9, 260, shortest=200)
    q, k, v, dy = tensors(1, 260, 4, 1, 64, dtype, factor=4.0)
    check(q, k, v, dy, spans)
    check(q, k, v, dy, spans, scale=0.01)
    check(q, k, v, dy, spans, scale=-0.25)
    # scores that fall by hundreds along the keys, and rise: the running maximum moves in every tile
    ramp = torch.linspace(-8, 8, 260, device="cuda").view(1, 260, 1, 1)
    for sign in (1, -1):
        check(torch.ones_like(q), (sign * ramp * torch.ones_like(k)).to(k.dtype), v, dy, spans, scale=1.0)


def test_no_documents_and_empty_batches():
    q, k, v, dy = tensors(2, 9, 4, 1, 64, "bf16")
    for value in run(q, k, v, dy, ()).values():
        assert (value == 0).all()
    for value in run(q, k, v, dy, ((0, 3, 3),)).values():
        assert (value == 0).all()
    for rows, width in ((0, 5), (2, 0)):
        assert run(*tensors(rows, width, 4, 1, 64, "bf16"), ())["y"].shape == (rows, width, 4, 64)


@pytest.mark.parametrize("dtype, heads, kv_heads, dim", [("bf16", 32, 1, 128), ("fp32", 4, 1, 64), ("fp16", 6, 3, 80)])
def test_repeated_calls_agree_bit_for_bit(dtype, heads, kv_heads, dim):
    spans = documents(2, 1500, 4, 1400)
    inputs = tensors(2, 1500, heads, kv_heads, dim, dtype)
    first, second = run(*inputs, spans), run(*inputs, spans)
    assert all(torch.equal(first[name], second[name]) for name in first)


def test_some_gradients_only():
    spans = documents(1, 100, 4, 60)
    q, k, v, dy = tensors(1, 100, 4, 1, 64, "bf16")
    plan = prepare_documents((1, 100), spans, "cuda", 4)
    everything = run(q, k, v, dy, spans)
    v.requires_grad_(True)
    y = document_attention(q, k, v, plan)
    assert torch.equal(torch.autograd.grad(y, v, dy)[0], everything["dv"])
    with torch.no_grad():
        assert torch.equal(document_attention(q, k, v, plan), everything["y"])


def test_gradients_against_differences():
    """<gradient, d> against central differences of the 64-bit formula along random directions."""
    spans = documents(1, 90, 4, 60, gap=4)
    q, k, v, dy = tensors(1, 90, 4, 2, 32, "fp32")
    actual = run(q, k, v, dy, spans)
    for index, name in enumerate(("dq", "dk", "dv")):
        direction = torch.randn_like((q, k, v)[index], dtype=torch.float64)
        step = 1e-5

        def value(sign):
            moved = [t.double() for t in (q, k, v)]
            moved[index] = moved[index] + sign * step * direction
            return float((reference(*moved, spans, 32 ** -0.5)[0]["y"] * dy.double()).sum())
        slope = (value(1) - value(-1)) / (2 * step)
        product = float((actual[name].double() * direction).sum())
        # fp32 gradients: 2^-24 relative each, sums of a few hundred terms; the difference itself is good to step^2
        size = float((actual[name].double().abs() * direction.abs()).sum())
        assert abs(product - slope) <= 1e-5 * size, name


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_on_another_stream_and_in_a_graph(dtype):
    spans = documents(2, 400, 4, 300, gap=3)
    q, k, v, dy = tensors(2, 400, 8, 1, 64, dtype)
    expected = run(q, k, v, dy, spans)
    plan = prepare_documents((2, 400), spans, "cuda", 8)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y, lse = attention_forward(q, k, v, plan)
        grads = attention_backward(dy, q, k, v, y, lse, plan)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip((y, *grads), expected.values()))
    # two captured graphs, replayed in turn with new inputs
    static = [t.clone() for t in (q, k, v, dy)]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, lse = attention_forward(*static[:3], plan)
            grads = attention_backward(static[3], *static[:3], y, lse, plan)
        graphs.append((graph, (y, *grads)))
    others = tensors(2, 400, 8, 1, 64, dtype, seed=5)
    expected_other = run(*others, spans)
    for inputs, results in (((q, k, v, dy), expected), (others, expected_other)):
        for target, source in zip(static, inputs):
            target.copy_(source)
        for graph, outputs in graphs:
            graph.replay()
        for graph, outputs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outputs, results.values()))


@pytest.mark.parametrize("heads, kv_heads", [(128, 1), (128, 128)])
def test_offsets_above_32_bits(heads, kv_heads):
    """More than 2^31 elements of q: the last documents come out as they do alone."""
    rows, width, dim = 137, 1024, 128
    assert rows * width * heads * dim > 2 ** 31
    generator = torch.Generator(device="cuda").manual_seed(3)
    make = lambda h: torch.randn(rows, width, h, dim, generator=generator, device="cuda", dtype=torch.bfloat16)
    q, k, v, dy = make(heads), make(kv_heads), make(kv_heads), make(heads)
    spans = tuple((row, start, start + 64) for row in range(rows) for start in range(0, width, 64))
    actual = run(q, k, v, dy, spans)
    for row in (0, rows - 1):
        alone = run(*(t[row:row + 1].clone() for t in (q, k, v, dy)), tuple((0, start, start + 64) for start in range(0, width, 64)))
        for name in ("y", "dq"):
            assert torch.equal(actual[name][row], alone[name][0]), name
        for name in ("dk", "dv"):             # pieces depend on the whole batch, so the order of sums does
            a, b = actual[name][row].double(), alone[name][0].double()
            assert float((a - b).norm()) <= 2.0 ** -8 * float(b.norm()), name


def test_two_host_threads_at_once():
    inputs = [tensors(2, 500, 8, 1, 64, "bf16", seed=i) for i in range(2)]
    spans = [documents(2, 500, i, 300, gap=3) for i in range(2)]
    expected = [run(*inputs[i], spans[i]) for i in range(2)]
    torch.cuda.synchronize()
    results = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                results[i] = run(*inputs[i], spans[i])
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    for i in range(2):
        assert all(torch.equal(results[i][name], expected[i][name]) for name in expected[i])


def test_a_plan_may_be_dropped_once_the_calls_are_issued():
    spans = documents(2, 700, 4, 300, gap=3)
    q, k, v, dy = tensors(2, 700, 8, 1, 64, "bf16")
    expected = run(q, k, v, dy, spans)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for _ in range(20):
        plan = prepare_documents((2, 700), spans, "cuda", 8)
        torch.cuda.current_stream().synchronize()
        with torch.cuda.stream(stream):
            y, lse = attention_forward(q, k, v, plan)
            grads = attention_backward(dy, q, k, v, y, lse, plan)
        records = plan.table.numel()
        del plan
        torch.full((records,), 7, device="cuda", dtype=torch.int32)       # where the table was, if it were given away
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((y, *grads), expected.values()))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_from_a_thread_that_has_not_used_cuda(dtype):
    spans = documents(1, 200, 4, 150)
    q, k, v, dy = tensors(1, 200, 4, 1, 64, dtype)
    plan = prepare_documents((1, 200), spans, "cuda", 4)
    y, lse = attention_forward(q, k, v, plan)
    expected = (y, *attention_backward(dy, q, k, v, y, lse, plan))
    torch.cuda.synchronize()
    results = {}
    forward = threading.Thread(target=lambda: results.update(forward=attention_forward(q, k, v, plan)))
    backward = threading.Thread(target=lambda: results.update(backward=attention_backward(dy, q, k, v, y, lse, plan)))
    for thread in (forward, backward):
        thread.start()
        thread.join()
    torch.cuda.synchronize()
    assert torch.equal(results["forward"][0], y) and torch.equal(results["forward"][1], lse)
    assert all(torch.equal(a, b) for a, b in zip(results["backward"], expected[1:]))


def test_refusals():
    q, k, v, dy = tensors(2, 20, 4, 1, 64, "bf16")
    plan = prepare_documents((2, 20), ((0, 0, 20),), "cuda", 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        document_attention(q.cpu(), k, v, plan)
    with pytest.raises(TypeError, match="one dtype"):
        document_attention(q, k.half(), v, plan)
    with pytest.raises(TypeError, match="libct_b200 supports"):
        document_attention(q.double(), k.double(), v.double(), plan)
    with pytest.raises(ValueError, match="the plan is for"):
        document_attention(q[:1], k[:1], v[:1], plan)
    with pytest.raises(ValueError, match="the plan is for"):
        document_attention(q[:, :, :2], k, v, plan)
    with pytest.raises(ValueError, match="document attention takes"):
        document_attention(q, k, v[..., :32], plan)
    with pytest.raises(ValueError, match="document attention takes"):
        document_attention(q.flatten(2), k, v, plan)
    with pytest.raises(NotImplementedError, match="head_dim"):
        document_attention(*(torch.zeros(2, 20, h, 136, device="cuda", dtype=torch.bfloat16) for h in (4, 1, 1)), plan)
    y, lse = attention_forward(q, k, v, plan)
    with pytest.raises(ValueError, match="shaped like q"):
        attention_backward(dy[:1], q, k, v, y, lse, plan)
    with pytest.raises(ValueError, match="lse"):
        attention_backward(dy, q, k, v, y, lse[:5], plan)
    with pytest.raises(ValueError, match="on one device"):
        document_attention(q, k, v, prepare_documents((2, 20), ((0, 0, 20),), "cpu", 4))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("heads, kv_heads", [(4, 1), (3, 3), (256, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_the_first_query_of_a_document_has_no_score_gradient(dtype, heads, kv_heads, dim):
    """It sees one key: P = 1 whatever its score, so dq is 0 for it, and dq and dk are for documents of one token."""
    q, k, v, dy = tensors(2, 150, heads, kv_heads, dim, dtype, factor=8.0)
    spans = ((0, 0, 1), (0, 1, 2), (0, 5, 140), (0, 140, 150), (1, 3, 4), (1, 4, 149), (1, 149, 150))
    grads = check(q, k, v, dy, spans)
    for row, start, end in spans:
        assert (grads["dq"][row, start] == 0).all()
        if end - start == 1:
            assert (grads["dk"][row, start] == 0).all() and (grads["dv"][row, start] != 0).any()
    dy[0, 1, 0, 0] = float("nan")                            # no zero hides it
    grads = run(q, k, v, dy, spans)
    assert torch.isnan(grads["dq"][0, 1, 0]).all() and torch.isnan(grads["dk"][0, 1, 0]).all() and torch.isnan(grads["dv"][0, 1, 0, 0])
    assert (grads["dq"][0, 1, 1:] == 0).all() and (grads["dq"][0, 0] == 0).all()
