"""Token embedding (kernels/embedding_cuda.py) against 64-bit values with derived bounds."""

import pytest
import torch

from causal_tuner_b200 import _lib
from causal_tuner_b200.kernels.embedding_cuda import embed_tokens, embedding_gradient, embedding_lookup

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_guard")]

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make_ids(tokens, rows, kind, seed=0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    u = torch.rand(tokens, generator=generator, device="cuda", dtype=torch.float64)
    ids = {"uniform": lambda: u * rows, "skewed": lambda: rows ** u - 1, "same": lambda: u * 0 + rows // 2,
           "two": lambda: (u > 0.3) * (rows - 1.0), "sorted": lambda: (u * rows).sort().values,
           "reverse": lambda: (u * rows).sort(descending=True).values}[kind]()
    return ids.long().clamp_(0, rows - 1)


def make_dy(tokens, width, dtype, seed=1):
    return torch.randn(tokens, width, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(TYPES[dtype])


@pytest.mark.parametrize("table", list(TYPES))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens, rows, width", [(1, 1, 1), (5, 97, 32), (77, 1000, 1001), (300, 513, 264), (0, 7, 8), (3, 7, 0)])
def test_lookup_is_one_rounding(table, dtype, tokens, rows, width):
    weight = make_dy(rows, width, table)
    ids = make_ids(tokens, rows, "uniform")
    for scale in (1.0, 16.0, 0.37):
        expected = (weight.float()[ids] * scale).to(TYPES[dtype])
        assert torch.equal(embedding_lookup(ids, weight, scale=scale, dtype=TYPES[dtype]), expected)
    assert embedding_lookup(ids, weight).dtype == weight.dtype


def check_gradient(ids, dy, rows, scale=1.0, padding_idx=None, dtype=torch.float32):
    """Sums in fp32 over n terms: n * 2^-24 of the sum of absolute values, the scale's product and the final rounding."""
    actual = embedding_gradient(dy, ids, rows, scale=scale, padding_idx=padding_idx, dtype=dtype)
    flat, wide = ids.flatten(), dy.reshape(-1, dy.shape[-1]).double()
    value = torch.zeros(rows, dy.shape[-1], device="cuda", dtype=torch.float64).index_add_(0, flat, wide)
    size = torch.zeros_like(value).index_add_(0, flat, wide.abs())
    count = torch.bincount(flat, minlength=rows).double().unsqueeze(1)
    e, u = 2.0 ** -24, torch.finfo(dtype).eps / 2
    if padding_idx is not None:
        value[padding_idx] = size[padding_idx] = 0
    value, bound = value * scale, abs(scale) * (count + 1) * e * size
    bound = bound + u * (value.abs() + bound)
    assert actual.dtype == dtype and actual.shape == (rows, dy.shape[-1])
    assert torch.isfinite(actual).all()
    assert float(((actual.double() - value).abs() - bound).max()) <= torch.finfo(dtype).smallest_normal if actual.numel() else True
    untouched = (count.squeeze(1) == 0)
    assert (actual[untouched] == 0).all()
    return actual


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["uniform", "skewed", "same", "two", "sorted", "reverse"])
@pytest.mark.parametrize("tokens, rows, width", [(1, 1, 1), (7, 97, 33), (128, 5, 32), (129, 300, 40), (1000, 1000, 256),
                                                 (1024, 5000, 8), (1025, 5000, 8), (4097, 70000, 24), (8193, 1 << 17, 8),
                                                 (16384, 3, 16), (16385, 300, 24), (32768, 70000, 8), (32769, 70000, 8), (40000, 1 << 17, 8)])
def test_gradient(dtype, kind, tokens, rows, width):
    check_gradient(make_ids(tokens, rows, kind), make_dy(tokens, width, dtype), rows)


@pytest.mark.parametrize("table", list(TYPES))
def test_gradient_scale_padding_and_table_types(table):
    ids, dy = make_ids(2000, 50, "skewed"), make_dy(2000, 72, "bf16")
    for padding_idx in (None, 0, 49, 3):
        actual = check_gradient(ids, dy, 50, scale=8.5, padding_idx=padding_idx, dtype=TYPES[table])
        if padding_idx is not None:
            assert (actual[padding_idx] == 0).all()
    assert torch.equal(embedding_gradient(dy, ids, 50, padding_idx=-1), embedding_gradient(dy, ids, 50, padding_idx=49))


def test_gradient_equals_the_sums_in_token_order():
    """Runs of up to 32 tokens are plain fp32 sums in token order: integers show that every token is counted once."""
    tokens, rows = 20000, 40000
    ids = make_ids(tokens, rows, "uniform")
    dy = torch.randint(-100, 100, (tokens, 16), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").float()
    expected = torch.zeros(rows, 16, device="cuda").index_add_(0, ids, dy)
    assert torch.equal(embedding_gradient(dy, ids, rows), expected)
    assert torch.equal(embedding_gradient(dy, ids.sort().values, rows), torch.zeros(rows, 16, device="cuda").index_add_(0, ids.sort().values, dy))


@pytest.mark.parametrize("tokens", [3000, 50000])
def test_gradient_is_reproducible(tokens):
    ids, dy = make_ids(tokens, 1000, "skewed"), make_dy(tokens, 64, "bf16")
    first = embedding_gradient(dy, ids, 1000)
    assert all(torch.equal(first, embedding_gradient(dy, ids, 1000)) for _ in range(3))


def test_layouts():
    """2-D ids of other integer types, strided and expanded gradients, a view at an odd address, no tokens at all."""
    ids, dy = make_ids(600, 90, "skewed"), make_dy(600, 48, "bf16")
    expected = embedding_gradient(dy, ids, 90)
    assert torch.equal(embedding_gradient(dy.view(20, 30, 48), ids.view(20, 30).int(), 90), expected)
    wide = torch.zeros(600, 100, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:51] = dy
    assert torch.equal(embedding_gradient(wide[:, 3:51], ids, 90), expected)
    assert torch.equal(embedding_gradient(dy.T.contiguous().T, ids, 90), expected)
    row = dy[:1].expand(600, 48)
    assert torch.equal(embedding_gradient(row, ids, 90), embedding_gradient(row.contiguous(), ids, 90))
    weight = make_dy(90, 48, "fp32")
    assert torch.equal(embedding_lookup(ids.view(20, 30).T, weight), weight[ids.view(20, 30).T])
    assert torch.equal(embedding_lookup(ids, weight.T.contiguous().T), weight[ids])
    odd = torch.zeros(90 * 48 + 1, device="cuda")[1:].view(90, 48)
    odd.copy_(weight)
    assert torch.equal(embedding_lookup(ids, odd), weight[ids])
    empty = ids[:0]
    assert (embedding_gradient(dy[:0], empty, 90) == 0).all() and embedding_lookup(empty, weight).shape == (0, 48)


def test_gradient_through_autograd_and_against_differences():
    ids = make_ids(200, 40, "skewed").view(10, 20)
    weight = make_dy(40, 24, "fp32").requires_grad_(True)
    dy = make_dy(200, 24, "fp32").view(10, 20, 24)
    out = embed_tokens(ids, weight, scale=3.0, padding_idx=2)
    grad, = torch.autograd.grad(out, weight, dy)
    direction = torch.randn(40, 24, device="cuda", dtype=torch.float64)
    direction[2] = 0
    value = lambda w: float((w[ids] * 3.0 * dy.double()).sum())
    slope = (value(weight.detach().double() + direction) - value(weight.detach().double() - direction)) / 2
    assert abs(float((grad.double() * direction).sum()) - slope) <= 1e-5 * float((grad.double().abs() * direction.abs()).sum())
    assert (grad[2] == 0).all()


def test_agrees_with_the_library_module():
    ids = make_ids(700, 300, "skewed").view(2, 350)
    module = torch.nn.Embedding(300, 64, padding_idx=5, device="cuda")
    dy = make_dy(700, 64, "bf16").view(2, 350, 64)
    expected = module(ids).to(torch.bfloat16)
    expected.backward(dy)
    out = embed_tokens(ids, module.weight, dtype=torch.bfloat16, padding_idx=module.padding_idx)
    assert torch.equal(out, expected)
    grad, = torch.autograd.grad(out, module.weight, dy)
    assert torch.allclose(grad, module.weight.grad, rtol=1e-4, atol=1e-4)


def test_ids_outside_the_table_are_reported():
    weight, dy = make_dy(10, 16, "fp32"), make_dy(4, 16, "fp32")
    ids = torch.tensor([3, 10, -1, 1 << 40], device="cuda")
    out = embedding_lookup(ids, weight)
    with pytest.raises(RuntimeError, match="outside the embedding table"):
        _lib.check_device()
    assert torch.equal(out[0], weight[3]) and (out[1:] == 0).all()
    grad = embedding_gradient(dy, ids, 10)
    with pytest.raises(RuntimeError, match="outside the embedding table"):
        _lib.check_device()
    assert torch.equal(grad[3], dy[0]) and float(grad.abs().sum()) == float(dy[0].abs().sum())
    _lib.check_device()


def test_on_another_stream_and_in_graphs():
    ids, dy, weight = make_ids(20000, 500, "skewed"), make_dy(20000, 64, "bf16"), make_dy(500, 64, "fp32")
    expected = embedding_lookup(ids, weight), embedding_gradient(dy, ids, 500)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        actual = embedding_lookup(ids, weight), embedding_gradient(dy, ids, 500)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(actual, expected))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = embedding_lookup(ids, weight), embedding_gradient(dy, ids, 500)
        graphs.append((graph, results))
    ids.copy_(make_ids(20000, 500, "uniform", seed=9))
    expected = embedding_lookup(ids, weight), embedding_gradient(dy, ids, 500)
    for graph, _ in graphs:
        graph.replay()
    for _, results in graphs:
        assert all(torch.equal(a, b) for a, b in zip(results, expected))


def test_offsets_above_32_bits():
    rows, width = (1 << 20) + 5, 2056
    assert rows * width > 2 ** 31
    weight = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
    ids = torch.tensor([rows - 1, 3, rows - 1, rows - 2, 0], device="cuda")
    weight[ids] = torch.arange(5 * width, device="cuda").view(5, width).remainder(200).to(torch.bfloat16)
    assert torch.equal(embedding_lookup(ids, weight), weight[ids])
    dy = make_dy(5, width, "bf16")
    grad = embedding_gradient(dy, ids, rows, dtype=torch.bfloat16)
    assert torch.equal(grad[rows - 1], (dy[0].float() + dy[2].float()).to(torch.bfloat16))
    assert torch.equal(grad[rows - 2], dy[3]) and torch.equal(grad[3], dy[1]) and torch.equal(grad[0], dy[4])
    assert int((grad != 0).any(1).sum()) == 4


def test_refusals():
    weight, ids, dy = make_dy(10, 16, "fp32"), make_ids(4, 10, "uniform"), make_dy(4, 16, "fp32")
    with pytest.raises(TypeError, match="integers"):
        embedding_lookup(ids.float(), weight)
    with pytest.raises(ValueError, match="matrix"):
        embedding_lookup(ids, weight[0])
    with pytest.raises(RuntimeError, match="no CPU path"):
        embedding_lookup(ids.cpu(), weight)
    with pytest.raises(TypeError, match="libct_b200 supports"):
        embedding_lookup(ids, weight.double())
    with pytest.raises(ValueError, match="one row per token"):
        embedding_gradient(dy[:3], ids, 10)
    with pytest.raises(ValueError, match="padding_idx"):
        embedding_gradient(dy, ids, 10, padding_idx=10)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("offset", [1, 2, 4, 8])
def test_results_at_any_element_of_a_buffer(dtype, offset):
    """The C entries take results that begin anywhere: 16 bytes past a 32-byte boundary is too little for the widest store."""
    tokens, rows, width = 37, 19, 24
    weight, ids, dy = make_dy(rows, width, dtype), make_ids(tokens, rows, "uniform"), make_dy(tokens, width, dtype, seed=2)
    library, code, stream = _lib.load(), _lib.code_of(TYPES[dtype]), _lib.stream_of(weight)
    buffer = torch.full((64 + tokens * width,), 7.0, device="cuda", dtype=TYPES[dtype])
    out = buffer[offset:offset + tokens * width]
    _lib.check(library.ct_embedding_forward(ids.data_ptr(), weight.data_ptr(), out.data_ptr(), tokens, rows, width, 1.0, code, code, stream))
    assert torch.equal(out.view(tokens, width), weight[ids])
    assert (buffer[:offset] == 7).all() and (buffer[offset + tokens * width:] == 7).all()
    buffer.fill_(7.0)
    table = buffer[offset:offset + rows * width]
    workspace = torch.empty(library.ct_embedding_gradient_workspace(tokens, rows, width), device="cuda", dtype=torch.uint8)
    _lib.check(library.ct_embedding_gradient(dy.data_ptr(), width, ids.data_ptr(), table.data_ptr(), tokens, rows, width, 1.0, -1, code, code,
                                             workspace.data_ptr(), stream))
    assert torch.equal(table.view(rows, width), embedding_gradient(dy, ids, rows, dtype=TYPES[dtype]))
    assert (buffer[:offset] == 7).all() and (buffer[offset + rows * width:] == 7).all()
