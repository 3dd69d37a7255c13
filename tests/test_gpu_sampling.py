"""GPU tests of sampling: tokens against the definition in 64 bits, equal but for nothing; log
probabilities to 2^-20, which counts FP32 exponentials of 2^-22 each and the rounding of the result."""
import importlib
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sampling(package):
    return importlib.import_module("nemotron_inference_b200.sampling")


def _token(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row, as the entry point's description says it."""
    x = x.astype(np.float64)
    top = x.max() if x.size else -np.inf
    if np.isnan(x).any() or not np.isfinite(top):
        return -1, math.nan
    logprob = lambda i: x[i] - top - math.log(math.fsum(np.exp(x - top)))  # noqa: E731
    if not temperature > 0:
        i = int(np.flatnonzero(x == top)[0])
        return i, logprob(i)
    order = np.argsort(-x, kind="stable")
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp(np.where(x[order] == -np.inf, -np.inf, (x[order] - top) / np.float64(np.float32(temperature))))
    w[np.isnan(w)] = 0.0
    if 1 <= top_k < x.size:
        order, w = order[:top_k], w[:top_k]
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        stay = before < float(np.float32(top_p)) * w.sum()
        stay[0] = True
        order, w = order[stay], w[stay]
    stay = w >= min(float(np.float32(min_p)), 1.0)
    order, w = order[stay], w[stay]
    rising = np.argsort(order)
    order, w = order[rising], w[rising]
    order, w = order[w > 0], w[w > 0]
    upto = np.cumsum(w)
    u = float(u) if u > 0 else 0.0
    at = int(np.searchsorted(upto, u * upto[-1], side="right"))
    i = int(order[min(at, order.size - 1)])
    return i, logprob(i)


def _check(sampling, logits, uniform, **parameters):
    tokens, logprobs = sampling.sample(logits, uniform, return_logprobs=True, **parameters)
    assert torch.equal(tokens, sampling.sample(logits, uniform, **parameters))
    x, u = logits.float().cpu().numpy(), uniform.cpu().numpy()
    tokens, logprobs = tokens.cpu().numpy(), logprobs.cpu().numpy()
    host = {k: v.cpu().numpy() if isinstance(v, torch.Tensor) else v for k, v in parameters.items() if v is not None}
    for i in range(x.shape[0]):
        of_row = {k: v[i] if isinstance(v, np.ndarray) else v for k, v in host.items()}
        token, logprob = _token(x[i], u[i], **of_row)
        assert tokens[i] == token, (i, tokens[i], token, of_row)
        if math.isnan(logprob):
            assert math.isnan(logprobs[i])
        else:
            assert abs(logprobs[i] - logprob) <= 2.0 ** -20 * max(1.0, abs(logprob)), (i, logprobs[i], logprob)


def _logits(rows, vocab, dtype, seed, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g, device="cuda") * spread
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 8), generator=g, device="cuda"),
                   torch.rand((rows, 8), generator=g, device="cuda") * 9.0)
    return x.to(dtype), torch.rand(rows, generator=g, device="cuda")


SETTINGS = [dict(), dict(temperature=0.7, top_p=0.95), dict(top_k=50), dict(temperature=1.3, top_k=700, top_p=0.8),
            dict(min_p=0.05), dict(temperature=0.0), dict(top_k=1), dict(temperature=0.9, top_k=40, top_p=0.9, min_p=0.1),
            dict(top_p=0.0), dict(top_p=0.999), dict(temperature=2.5, top_p=0.7)]


@pytest.mark.parametrize("rows,vocab", [(1, 131072), (3, 1), (2, 2), (70, 7), (5, 33), (40, 1000), (9, 50001),
                                        (160, 4099), (2, 262144), (1, 393216)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens(sampling, rows, vocab, dtype):
    for number, setting in enumerate(SETTINGS):
        logits, uniform = _logits(rows, vocab, dtype, 100 * number + rows)
        _check(sampling, logits, uniform, **setting)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [3001, 70000])
def test_parameters_of_each_row(sampling, vocab, dtype):
    rows = 48
    logits, uniform = _logits(rows, vocab, dtype, 5)
    rng = np.random.default_rng(6)
    vector = lambda values, kind: torch.tensor(rng.choice(values, rows), dtype=kind, device="cuda")  # noqa: E731
    _check(sampling, logits, uniform, temperature=vector([0.0, -1.0, 0.3, 1.0, 1.7], torch.float32),
           top_k=vector([-3, 0, 1, 2, 300, 2 ** 31 - 1], torch.int32),
           top_p=vector([0.0, 0.1, 0.9, 1.0, 2.0], torch.float32), min_p=vector([0.0, 0.01, 1.0, 3.0], torch.float32))


@pytest.mark.parametrize("vocab", [5, 300, 1000, 131072])
def test_equal_logits(sampling, vocab):
    """All tokens weigh the same: sums are whole numbers, so each token's share is known exactly."""
    logits = torch.full((33, vocab), -2.25, device="cuda")
    uniform = torch.arange(33, device="cuda") / 33.0
    for setting in (dict(), dict(top_k=4), dict(top_k=vocab // 2 + 1), dict(top_p=0.5), dict(top_p=0.9, top_k=vocab - 1),
                    dict(min_p=1.0), dict(temperature=0.0)):
        _check(sampling, logits, uniform, **setting)


def test_few_values(sampling):
    """Hundreds of tokens share each value, so borders lie inside such groups."""
    logits, uniform = _logits(24, 60000, torch.float32, 8)
    logits = (logits * 2).round() / 2
    logits[:, ::7] *= -0.0  # both zeros are one value
    for setting in (dict(top_k=2000), dict(top_p=0.97), dict(temperature=1.5, top_k=30000, top_p=0.9), dict(temperature=0.0)):
        _check(sampling, logits, uniform, **setting)


def test_many_values_close_together(sampling):
    """A whole vocabulary within one bin of the histogram."""
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = 5.0 + 0.01 * torch.rand((6, 90000), generator=g, device="cuda")
    uniform = torch.rand(6, generator=g, device="cuda")
    for setting in (dict(top_k=33333), dict(top_p=0.5), dict(top_k=70000, top_p=0.25), dict()):
        _check(sampling, logits, uniform, **setting)
    around_zero = (logits - 5.005) * 1e-20  # (their bits lie far apart)
    for setting in (dict(top_k=33333), dict(top_p=0.5)):
        _check(sampling, around_zero, uniform, **setting)


def test_many_rows_of_values_close_together(sampling):
    """One block to a row, and more tokens near the border than it notes."""
    g = torch.Generator(device="cuda").manual_seed(3)
    logits, uniform = _logits(72, 131072, torch.float32, 17, spread=1.0)
    close = 1.0 + 1e-3 * torch.rand(logits.shape, generator=g, device="cuda")
    logits = torch.where(torch.rand(logits.shape, generator=g, device="cuda") < 0.6, close, logits)
    for setting in (dict(top_p=0.6), dict(top_k=40000), dict(top_k=90000, top_p=0.5)):
        _check(sampling, logits, uniform, **setting)


@pytest.mark.parametrize("rows", [2, 80])
def test_borders_among_few_heavy_tokens(sampling, rows):
    """What most of a row's tokens say about the border is wrong: a few others weigh as much as all of them."""
    g = torch.Generator(device="cuda").manual_seed(4)
    logits, uniform = _logits(rows, 131072, torch.float32, 18, spread=1.0)
    logits = logits.clamp(max=4.0)
    heavy = torch.rand((rows, 40), generator=g, device="cuda") * 8.0 + torch.linspace(2.0, 9.0, rows, device="cuda")[:, None]
    logits.scatter_(1, torch.randint(0, 131072, (rows, 40), generator=g, device="cuda"), heavy)
    for top_p in (0.3, 0.8, 0.95, 0.99, 0.999):
        _check(sampling, logits, uniform, top_p=top_p)
    _check(sampling, logits, uniform, top_k=300, top_p=0.99, temperature=1.4)


def test_large_batch(sampling):
    rows = 150
    logits, uniform = _logits(rows, 131072, torch.bfloat16, 19)
    rng = np.random.default_rng(20)
    vector = lambda values, kind: torch.tensor(rng.choice(values, rows), dtype=kind, device="cuda")  # noqa: E731
    _check(sampling, logits, uniform, temperature=vector([0.0, 0.5, 1.0, 1.6], torch.float32),
           top_k=vector([0, 0, 20, 300, 20000], torch.int32), top_p=vector([0.5, 0.95, 0.999, 1.0], torch.float32),
           min_p=vector([0.0, 0.0, 0.02], torch.float32))


def test_masks(sampling):
    logits, uniform = _logits(12, 20000, torch.float32, 9)
    lowest = torch.finfo(torch.float32).min
    logits[0] = -math.inf                       # nothing left
    logits[1, 5] = math.nan
    logits[2, 7] = math.inf
    logits[3] = lowest                          # all masked by the lowest value: equal ones
    logits[4] = -math.inf
    logits[4, 19999] = -3.0                     # one left
    logits[5, 1:] = lowest
    logits[6, :19000] = -math.inf
    logits[7] = -math.inf
    logits[7, 100] = logits[7, 300] = lowest    # the largest is the lowest
    logits[8] = 3e38
    logits[9, 3] = 3.4e38
    logits[10] = -math.nan
    for setting in SETTINGS:
        _check(sampling, logits, uniform, **setting)


@pytest.mark.parametrize("temperature", [1e-38, 1e-45, 1e-6, 1e6, 3e38, math.inf])
def test_temperatures_at_the_ends(sampling, temperature):
    logits, uniform = _logits(6, 5000, torch.float32, 10)
    logits[:, 17] = -math.inf
    logits[2, 40] = logits[2, 41] = 30.0
    for setting in (dict(), dict(top_k=20), dict(top_p=0.5), dict(min_p=0.5)):
        _check(sampling, logits, uniform, temperature=temperature, **setting)


def test_random_numbers_at_the_ends(sampling):
    values = [0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan, 1e-30, math.inf]
    logits, _ = _logits(len(values), 4000, torch.float32, 11)
    uniform = torch.tensor(values, device="cuda")
    for setting in (dict(), dict(top_k=3), dict(top_p=0.9)):
        tokens = sampling.sample(logits, uniform, **setting)
        inside = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0 - 2.0 ** -24, 1.0 - 2.0 ** -24, 0.0, 0.0, 1e-30, 1.0 - 2.0 ** -24],
                              device="cuda")
        last = sampling.sample(logits, inside, **setting)
        assert torch.equal(tokens[[0, 4, 5, 6]], last[[0, 4, 5, 6]])
        _check(sampling, logits, inside, **setting)
        for i in (2, 3, 7):  # the last one that stays
            x = logits[i].cpu().numpy()
            assert tokens[i] == _token(x, 1.0, **setting)[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first,vocab,stride", [(1, 1001, 1007), (3, 30000, 30011), (0, 50001, 50048), (5, 6, 13)])
def test_rows_that_begin_anywhere(sampling, first, vocab, stride, dtype):
    whole, uniform = _logits(7, stride, dtype, 12)
    whole[:, :first] = 100.0        # what lies beside a row is not part of it
    whole[:, first + vocab:] = math.nan
    for setting in (dict(temperature=0.8, top_p=0.9), dict(top_k=5), dict(temperature=0.0)):
        _check(sampling, whole[:, first:first + vocab], uniform, **setting)


def test_a_row_does_not_depend_on_its_batch(sampling):
    logits, uniform = _logits(300, 40000, torch.float32, 13, spread=0.5)
    together, of_all = sampling.sample(logits, uniform, top_p=0.9, return_logprobs=True)
    for i in (0, 7, 299):
        alone, of_one = sampling.sample(logits[i:i + 1], uniform[i:i + 1], top_p=0.9, return_logprobs=True)
        assert alone[0] == together[i]
        assert abs(of_one[0] - of_all[i]) <= 2.0 ** -20 * max(1.0, float(of_all[i].abs()))
    again, of_again = sampling.sample(logits, uniform, top_p=0.9, return_logprobs=True)
    assert torch.equal(again, together) and torch.equal(of_again, of_all)


def test_recorded_and_on_another_stream(sampling):
    logits, uniform = _logits(16, 33000, torch.float32, 14)
    top_p = torch.full((16,), 0.9, device="cuda")
    out = torch.empty(16, dtype=torch.int32, device="cuda")
    sampling.sample(logits, uniform, top_p=top_p, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sampling.sample(logits, uniform, top_p=top_p, out=out)
    more, numbers = _logits(16, 33000, torch.float32, 15)
    logits.copy_(more)
    uniform.copy_(numbers)
    top_p.fill_(0.6)
    graph.replay()
    replayed = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = sampling.sample(more, numbers, top_p=0.6)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(replayed, aside)
    _check(sampling, more, numbers, top_p=0.6)


def test_more_rows_than_a_grid_dimension_has_blocks(sampling):
    rows = 70000
    logits, uniform = _logits(rows, 50, torch.float32, 21)
    assert torch.equal(sampling.sample(logits, uniform, temperature=0.0).long(), logits.argmax(1))
    tokens, logprobs = sampling.sample(logits, uniform, temperature=0.8, top_k=20, top_p=0.9, return_logprobs=True)
    x, u = logits.cpu().numpy(), uniform.cpu().numpy()
    for i in (0, 1, 65535, 65536, rows - 1):
        token, logprob = _token(x[i], u[i], temperature=0.8, top_k=20, top_p=0.9)
        assert tokens[i] == token
        assert abs(float(logprobs[i]) - logprob) <= 2.0 ** -20 * max(1.0, abs(logprob))


def test_two_calls_on_two_streams_and_in_two_graphs(sampling):
    one, of_one = _logits(40, 70000, torch.float32, 22)
    two, of_two = _logits(90, 50001, torch.bfloat16, 23)
    want = sampling.sample(one, of_one, top_p=0.9), sampling.sample(two, of_two, top_k=500, top_p=0.95)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    graphs, outs = [], []
    for stream, logits, uniform, setting in ((streams[0], one, of_one, dict(top_p=0.9)),
                                             (streams[1], two, of_two, dict(top_k=500, top_p=0.95))):
        out = torch.zeros(logits.shape[0], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            sampling.sample(logits, uniform, out=out, **setting)
        graphs.append(graph)
        outs.append(out)
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    with torch.cuda.stream(streams[0]):
        again = sampling.sample(one, of_one, top_p=0.9)
    with torch.cuda.stream(streams[1]):
        and_again = sampling.sample(two, of_two, top_k=500, top_p=0.95)
    torch.cuda.synchronize()
    for got, expected in zip(outs + [again, and_again], want + want):
        assert torch.equal(got, expected)


def test_refusals(sampling, package):
    logits, uniform = _logits(4, 100, torch.float32, 16)
    for bad in (dict(logits=logits.half()), dict(logits=logits[0]), dict(logits=logits.t()), dict(uniform=uniform[:3]),
                dict(uniform=uniform.double()), dict(temperature=uniform[:2]), dict(top_k=uniform), dict(top_k=1.5),
                dict(temperature=math.nan), dict(top_p=math.nan), dict(min_p=math.nan), dict(logits=logits.cpu()),
                dict(logits=logits[:1].expand(4, 100)), dict(out=torch.empty(4, device="cuda")), dict(uniform=uniform.cpu()),
                dict(logits=logits[:, :0])):
        arguments = dict(logits=logits, uniform=uniform)
        arguments.update(bad)
        with pytest.raises(ValueError):
            sampling.sample(**arguments)
    with pytest.raises(package.NmoeError) as info:
        sampling.sample(torch.zeros((1, 393217), device="cuda"), uniform[:1])
    assert info.value.status == 3
    assert sampling.sample(logits[:0], uniform[:0]).numel() == 0
