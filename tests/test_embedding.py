"""Token embedding: lookup and table gradient against FP64 sums, from one token
to runs that span many chunks, and refusals."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from lsso_amd.ball import TokenEmbedding, hip
from lsso_amd.ball import reference as canonical

TYPES = (torch.float16, torch.bfloat16, torch.float32)


def test_module_on_the_cpu() -> None:
    layer = TokenEmbedding(6, 4, scale=2.0, padding_index=1)
    tokens = torch.tensor([[0, 1, 5], [3, 3, 99]])
    mask = torch.tensor([[True, True, True], [True, True, False]])
    y = layer(tokens, mask)
    assert torch.equal(y[0, 2], 2 * layer.weight[5]) and torch.equal(y[1, 2], torch.zeros(4))
    y.sum().backward()
    assert torch.equal(layer.weight.grad[:, 0], torch.tensor([2.0, 0, 0, 4, 0, 2]))
    assert layer(tokens[:1], dtype=torch.float64).dtype == torch.float64
    for wrong in ({"vocabulary": 0}, {"padding_index": 6}):
        with pytest.raises(ValueError):
            TokenEmbedding(**{"vocabulary": 6, "dim": 4, **wrong})


def test_refusals_on_the_cpu() -> None:
    library = hip.open_library()
    size = ctypes.c_size_t()

    def lookup(tokens=16, wide=8, count=4, weight=16, kind=2, vocabulary=9, dim=8, stride=8, mask=None, y=16, out=2):
        return library.lsso_hip_embedding(tokens, wide, count, weight, kind, vocabulary, dim, stride, 1.0, mask, y, out,
                                          None)

    def grad(count=4, dy=16, kind=2, stride=8, vocabulary=9, dim=8, padding=-1, out=16, weight=2, workspace=256,
             room=1 << 20):
        return library.lsso_hip_embedding_grad(16, 8, count, dy, kind, stride, vocabulary, dim, 1.0, None, padding, out,
                                               weight, workspace, room, None)

    assert lookup(count=0, tokens=None, weight=None, y=None) == 0
    for wrong in ({"count": -1}, {"count": 2**31}, {"vocabulary": 0}, {"dim": 0}, {"dim": 2**25}, {"wide": 2},
                  {"tokens": None}, {"tokens": 12}, {"kind": 0}, {"out": 9}, {"stride": 7}, {"weight": None},
                  {"y": 17}, {"vocabulary": 2**31}):
        assert lookup(**wrong) < 0, wrong
    for wrong in ({"count": -1}, {"kind": 7}, {"weight": 0}, {"stride": 7}, {"padding": 9}, {"padding": -2},
                  {"out": None}, {"dy": None}, {"workspace": None}, {"workspace": 128}, {"room": 64}):
        assert grad(**wrong) < 0, wrong
    assert library.lsso_hip_embedding_grad_workspace_bytes(4, 9, 8, None) < 0
    assert library.lsso_hip_embedding_grad_workspace_bytes(4, 0, 8, ctypes.byref(size)) < 0
    assert library.lsso_hip_embedding_grad_workspace_bytes(2**31 - 1, 2**31 - 2, 8, ctypes.byref(size)) == 0
    assert size.value > 16 * 2**31   # two copies of ids and indices: no 32-bit size


def _tokens(kind, count, vocabulary, generator):
    if kind == "uniform":
        return torch.randint(0, vocabulary, (count,), generator=generator)
    if kind == "one":
        return torch.full((count,), vocabulary // 2)
    u = torch.rand(count, generator=generator, dtype=torch.float64)
    return torch.exp(u * math.log(vocabulary + 1.0)).sub(1).long().clamp(0, vocabulary - 1)


def _check(native, tokens, vocabulary, dim, table, out, mask=None, padding=None, scale=3.25):
    generator = torch.Generator().manual_seed(5)
    weight = torch.randn(vocabulary, dim, generator=generator).to(table)
    dy = torch.randn(*tokens.shape, dim, generator=generator).to(out)
    wd = weight.cuda().requires_grad_()
    y = native.embedding(tokens.cuda(), wd, scale=scale, row_mask=None if mask is None else mask.cuda(),
                         padding_index=padding, output_dtype=out)
    named = torch.where((tokens >= 0) & (tokens < vocabulary), tokens, 0).long()
    kept = torch.ones_like(tokens, dtype=torch.bool) if mask is None else mask
    outside = (named != tokens) & kept
    expected = scale * weight.double()[named]
    expected[~kept] = 0.0
    expected[outside] = math.nan
    assert y.shape == expected.shape and y.dtype == out and y.is_contiguous()
    half = torch.finfo(out).eps / 2
    got = y.detach().cpu().double()
    assert torch.equal(got.isnan(), expected.isnan())
    # scale is exact in FP32: one rounding of the product and one to the type.
    limit = (half + 2.0**-23) * expected.abs() + 2.0**-25
    assert ((got - expected).abs() <= limit)[~expected.isnan()].all()
    (grad,) = torch.autograd.grad(y, (wd,), dy.cuda())
    again = torch.autograd.grad(
        native.embedding(tokens.cuda(), wd, scale=scale, row_mask=None if mask is None else mask.cuda(),
                         padding_index=padding, output_dtype=out), (wd,), dy.cuda())[0]
    assert torch.equal(grad, again)
    counted = kept & (named == tokens)
    if padding is not None:
        counted &= tokens != padding
    rows, ids = dy.double()[counted], tokens[counted].long()
    expected = torch.zeros(vocabulary, dim, dtype=torch.float64).index_add_(0, ids, rows) * scale
    absolute = torch.zeros(vocabulary, dim, dtype=torch.float64).index_add_(0, ids, rows.abs()) * scale
    # n - 1 FP32 additions in any order, the product with the scale, the type.
    n = torch.bincount(ids, minlength=vocabulary).clamp_min(1)[:, None]
    half = torch.finfo(table).eps / 2
    limit = n * 2.0**-24 * absolute * 1.01 + (half + 2.0**-23) * expected.abs() + 2.0**-25
    assert grad.dtype == table
    got = grad.cpu().double()
    assert ((got - expected).abs() <= limit).all()
    assert (got[torch.bincount(ids, minlength=vocabulary) == 0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("table", TYPES)
@pytest.mark.parametrize("out", TYPES)
def test_types(native, table, out) -> None:
    generator = torch.Generator().manual_seed(2)
    _check(native, _tokens("uniform", 197, 37, generator).view(1, 197), 37, 40, table, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", (1, 7, 8, 9, 64, 100, 301, 512, 521, 1030))
@pytest.mark.parametrize("kind", ("uniform", "one"))
def test_widths(native, dim, kind) -> None:
    generator = torch.Generator().manual_seed(3)
    _check(native, _tokens(kind, 300, 5, generator).view(3, 100), 5, dim, torch.bfloat16, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("count", (1, 2, 63, 64, 65, 129, 4095, 4097, 20000))
@pytest.mark.parametrize("vocabulary", (1, 2, 6, 257, 1023, 1024, 1025, 40000))
def test_counts_and_vocabularies(native, count, vocabulary) -> None:
    generator = torch.Generator().manual_seed(count + vocabulary)
    kind = "uniform" if vocabulary < 100 else "skewed"
    _check(native, _tokens(kind, count, vocabulary, generator), vocabulary, 24, torch.float32, torch.float16)


@pytest.mark.gpu
def test_many_tokens(native) -> None:
    generator = torch.Generator().manual_seed(8)
    # Tiles, chunk lengths and passes of a large batch; runs of 60,000 tokens.
    _check(native, _tokens("uniform", 300001, 5, generator), 5, 16, torch.float32, torch.bfloat16)
    _check(native, _tokens("skewed", 600011, 1200000, generator), 1200000, 8, torch.float16, torch.float16)
    _check(native, _tokens("one", 1100000, 3, generator), 3, 8, torch.float32, torch.float32)


@pytest.mark.gpu
def test_runs_at_chunk_borders(native) -> None:
    # Runs of 64 and 65 tokens (chunks of 32: added whole, by chunks) that
    # begin at, before and behind a chunk's border.
    for lengths in ((64, 65, 64), (65, 65, 65), (31, 65, 1, 64, 66), (32, 96, 96), (1, 127, 65, 33, 200), (95, 97)):
        tokens = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
        shuffle = torch.randperm(tokens.numel(), generator=torch.Generator().manual_seed(1))
        _check(native, tokens[shuffle], len(lengths), 16, torch.float32, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("count,chunk", [(32767, 16), (32768, 32), (98303, 32), (98304, 64), (524287, 64), (524288, 128)])
def test_runs_at_the_borders_of_every_chunk_length(native, count, chunk) -> None:
    """Runs that end before, at and behind a chunk's border, from a chunk's length
    to more than a wave joins (16 chunks), each then a run of the rest."""

    lengths = [chunk - 1, 1, chunk, chunk + 1, chunk - 1, 2 * chunk, 1, 15 * chunk - 2, chunk + 2, 16 * chunk,
               16 * chunk + 1, chunk - 1, 33 * chunk, 3]
    lengths.append(count - sum(lengths))
    tokens = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
    shuffle = torch.randperm(count, generator=torch.Generator().manual_seed(3))
    _check(native, tokens[shuffle], len(lengths), 8, torch.float32, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", (5, 16, 520))
def test_runs_inside_chunks_across_them_and_joined(native, dim) -> None:
    # Runs that end inside a chunk of 16, cross its ends, and are joined by a wave
    # (up to 16 chunks) or a workgroup.
    for lengths in ((8, 9, 7, 8, 10, 8), (30, 8, 30, 9, 30, 4), (31, 1, 8, 24, 9, 9), (16 * 16, 1, 16 * 16 + 1),
                    (10, 15 * 16 + 6, 5), (10, 15 * 16 + 7, 5), (16 * 32, 1, 16 * 32 + 1),
                    (20, 15 * 32 + 12, 5), (20, 15 * 32 + 13, 5), (3, 17 * 32, 40, 70 * 32 + 5, 1)):
        tokens = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
        shuffle = torch.randperm(tokens.numel(), generator=torch.Generator().manual_seed(2))
        _check(native, tokens[shuffle], len(lengths) + 1, dim, torch.float32, torch.float32)


@pytest.mark.gpu
def test_offsets_past_32_bits(native) -> None:
    count, dim = 262200, 8200
    weight = torch.randn(5, dim, device="cuda").bfloat16().requires_grad_()
    tokens = torch.arange(count, device="cuda") % 5
    y = native.embedding(tokens, weight)
    assert torch.equal(y[-7:], weight.detach()[tokens[-7:]])
    dy = torch.zeros_like(y)
    dy[-7:] = torch.randint(-8, 9, (7, dim), device="cuda")   # sums of small integers are exact
    (grad,) = torch.autograd.grad(y, weight, dy)
    expected = torch.zeros(5, dim, device="cuda").index_add_(0, tokens[-7:], dy[-7:].float())
    assert torch.equal(grad.float(), expected)


@pytest.mark.gpu
def test_tables_past_one_launch_of_eight_rows_a_wave(native) -> None:
    vocabulary = (1 << 29) + 77
    weight = torch.zeros(vocabulary, 1, dtype=torch.bfloat16, device="cuda")
    tokens = torch.tensor([3, vocabulary - 1, 1 << 28, vocabulary - 1, vocabulary, 0], device="cuda")
    weight[tokens[1]] = 5.0
    weight.requires_grad_()
    y = native.embedding(tokens, weight)
    assert y[1].item() == y[3].item() == 5.0 and y[0].item() == 0.0 and y[4].isnan().all()
    (grad,) = torch.autograd.grad(y, weight, torch.full_like(y, 1.5))
    named = grad.nonzero()[:, 0]
    assert named.tolist() == [0, 3, 1 << 28, vocabulary - 1]
    assert grad[named, 0].tolist() == [1.5, 1.5, 1.5, 3.0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.int32, torch.int64))
def test_masks_padding_and_ids_outside(native, dtype) -> None:
    generator = torch.Generator().manual_seed(4)
    tokens = torch.randint(0, 11, (4, 50), generator=generator).to(dtype)
    mask = torch.rand(4, 50, generator=generator) < 0.6
    mask[2] = False
    tokens[~mask] = -100
    tokens[0, 3], tokens[1, 7], tokens[3, 0] = 11, -1, torch.iinfo(dtype).max
    mask[0, 3] = mask[1, 7] = mask[3, 0] = True
    _check(native, tokens, 11, 33, torch.float32, torch.bfloat16, mask=mask, padding=4)
    _check(native, tokens.clamp(0, 10), 11, 33, torch.float32, torch.bfloat16, mask=torch.zeros_like(mask))
    # Excluded gradients may hold anything.
    weight = torch.randn(11, 8, device="cuda", requires_grad=True)
    keep = torch.tensor([True, False, True], device="cuda")
    y = native.embedding(torch.tensor([1, 1, 2], device="cuda"), weight, row_mask=keep, padding_index=2)
    dy = torch.ones_like(y)
    dy[1:] = math.nan
    (grad,) = torch.autograd.grad(y, weight, dy)
    assert torch.equal(grad[1], torch.ones(8, device="cuda")) and not grad[2:].any() and not grad[0].any()


@pytest.mark.gpu
def test_views_and_empty_batches(native) -> None:
    table = torch.randn(40, 30, device="cuda")
    view = table[3:23, 1:18].requires_grad_()   # rows and base aligned to one element
    tokens = torch.randint(0, 20, (6, 10), device="cuda")
    assert torch.equal(native.embedding(tokens.t(), view), view.detach()[tokens.t()])
    dy = torch.randn(10, 6, 17, device="cuda").transpose(0, 1)
    (grad,) = torch.autograd.grad(native.embedding(tokens, view), view, dy)
    expected = torch.zeros(20, 17, dtype=torch.float64, device="cuda").index_add_(
        0, tokens.reshape(-1), dy.reshape(-1, 17).double())
    torch.testing.assert_close(grad.double(), expected, rtol=1e-5, atol=1e-5)
    (grad,) = torch.autograd.grad(native.embedding(tokens, view).sum(), view)   # stride-0 gradient
    assert torch.equal(grad[:, 0], torch.bincount(tokens.reshape(-1), minlength=20).float())
    y = native.embedding(tokens[:0], view)
    assert y.shape == (0, 10, 17)
    (grad,) = torch.autograd.grad(y.sum(), view)
    assert grad.shape == (20, 17) and not grad.any()


@pytest.mark.gpu
def test_captured_training_step(native) -> None:
    weight = torch.randn(1500, 48, device="cuda", requires_grad=True)
    tokens = torch.randint(0, 1500, (700,), device="cuda")
    dy = torch.randn(700, 48, device="cuda")

    def step():
        y = native.embedding(tokens, weight, scale=2.0)
        return y.detach(), torch.autograd.grad(y, weight, dy)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, grad = step()
    for replay in range(3):
        tokens.copy_(torch.randint(0, 3 if replay == 1 else 1500, (700,), device="cuda"))
        dy.normal_()
        graph.replay()
        expected = step()
        assert torch.equal(y, expected[0]) and torch.equal(grad, expected[1])


@pytest.mark.gpu
def test_refusals(native) -> None:
    weight = torch.randn(5, 8, device="cuda")
    tokens = torch.zeros(3, dtype=torch.int64, device="cuda")
    for arguments, options, error in (
        ((tokens, weight.cpu()), {}, RuntimeError), ((tokens.cpu(), weight), {}, RuntimeError),
        ((tokens.float(), weight), {}, TypeError), ((tokens, weight.double()), {}, TypeError),
        ((tokens, weight[0]), {}, TypeError), ((tokens, weight[:0]), {}, ValueError),
        ((tokens, weight), {"padding_index": 5}, ValueError), ((tokens, weight), {"padding_index": -1}, ValueError),
        ((tokens, weight), {"row_mask": torch.ones(2, dtype=torch.bool, device="cuda")}, ValueError),
        ((tokens, weight), {"row_mask": tokens}, ValueError), ((tokens, weight), {"output_dtype": torch.float64}, TypeError),
        ((tokens, weight), {"row_mask": torch.ones(3, dtype=torch.bool)}, RuntimeError),
    ):
        with pytest.raises(error):
            native.embedding(*arguments, **options)


@pytest.mark.gpu
def test_module_paths_agree(native) -> None:
    layer = TokenEmbedding(20, 24, scale=2.0, padding_index=3)
    tokens = torch.randint(0, 20, (4, 9))
    mask = torch.rand(4, 9) < 0.7
    layer(tokens, mask).square().sum().backward()
    expected = layer.weight.grad.clone()
    layer.weight.grad = None
    layer.cuda()
    layer(tokens.cuda(), mask.cuda(), implementation="hip").square().sum().backward()
    torch.testing.assert_close(layer.weight.grad.cpu(), expected, rtol=1e-5, atol=1e-5)
    assert canonical.embedding(tokens, layer.weight.detach().cpu()).shape == (4, 9, 24)
