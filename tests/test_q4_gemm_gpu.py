"""linear_q4 in sizes that take the tensor-core GEMM (above 32 tokens about twice the size where the choice falls on
it): every test looks whether it ran, by the launches it takes (the preparation of the scales and the GEMM;
copied rows add one launch for the weights and one for the tokens).

Integer cases have products and partial sums that are exact in fp32 and in fp16 up to the last rounding, so a wrong
index, scale, mask or join of partial sums changes bits.
"""
import warnings

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _weights(cuda, N, K, group, seed, exps=(-2, 1)):
    """Random codes, scales of random powers of two, and the values in 64 bits."""
    import torch

    g = torch.Generator(device=cuda).manual_seed(seed)
    q4 = torch.randint(0, 256, (N, (K + 1) // 2), dtype=torch.uint8, device=cuda, generator=g)
    if K % 2:
        q4[:, -1] = (q4[:, -1] & 15) | 0x80
    sc = (2.0 ** torch.randint(*exps, (N, -(-K // group)), device=cuda, generator=g)).bfloat16()
    return q4, sc


def _values(q4, sc, K, group):
    import torch

    q = torch.stack((q4 & 15, q4 >> 4), dim=-1).flatten(1)[:, :K].double() - 8
    return q * sc.double().repeat_interleave(group, dim=1)[:, :K]


def _tokens(cuda, M, K, seed):
    import torch

    return torch.randint(-3, 4, (M, K), device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)).half()


def _gemm(out, x, q4, sc, group, bias=None, residual=None, stream=None):
    """The call, and that it was the GEMM: two launches, or with copied rows four (aligned tensors here)."""
    import vvllm_b200 as v

    before = v.launch_count()
    v.linear_q4_add(out, x, q4, sc, group, bias, residual, stream=stream)
    if v.launch_count() - before != (2 if x.shape[1] % 32 == 0 else 4):
        said = f"{list(x.shape)} x {q4.shape[0]} rows did not take the GEMM"
        assert len(x) <= 32, said  # up to there the choice is close
        warnings.warn(said)


# Token tiles of 16, 32, 64, 128 and 256 (300 tokens: 32-, 128- and 256-wide by the number of row tiles), rows that end
# within a stage, more than 160 groups of 32 to a row, row counts that allow vector stores and that do not.
CASES = [(9, 2700, 22784), (12, 2601, 18976), (16, 2504, 18944), (17, 15001, 1056), (24, 10704, 1056), (32, 8503, 1056),
         (33, 16000, 1056), (48, 9000, 5184), (64, 7003, 5216), (65, 8000, 1056), (100, 5203, 1056), (128, 5000, 3616),
         (129, 4008, 1056), (300, 1701, 5216), (300, 2000, 1056), (300, 5003, 1056), (512, 904, 5184)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", CASES)
def test_exact_on_integers(cuda, M, N, K, group):
    import torch

    import vvllm_b200 as v

    q4, sc = _weights(cuda, N, K, group, M + K)
    x = _tokens(cuda, M, K, N)
    y = x.double() @ _values(q4, sc, K, group).T
    assert y.abs().max() < 2 ** 15  # fp16 holds it, fp32 its quarters
    r = np.random.default_rng(M)
    bias = torch.from_numpy(r.integers(-50, 50, N)).to(cuda).float()
    res = torch.from_numpy(r.integers(-50, 50, (M, N))).to(cuda).half()
    for b, in_place in ((None, False), (bias, False), (bias, True), (None, True)):
        guard = torch.full((M + 2, N), 77.0, dtype=torch.float16, device=cuda)
        out = guard[1:M + 1] if N % 8 else guard[1:M + 1].clone()
        residual, want = None, y if b is None else y + b.double()
        if in_place:
            out.copy_(res)
            residual, want = out, want + res.double()
        _gemm(out, x, q4, sc, group, b, residual)
        assert torch.equal(out, want.half()), (b is None, in_place)
        assert (guard[0] == 77).all() and (guard[-1] == 77).all()
    assert v.kernel_error() == 0


@pytest.mark.parametrize("M,N,K", [(24, 22003, 512), (48, 22000, 512), (100, 11003, 480), (300, 3600, 512), (700, 12000, 96)])
def test_fp32_outputs_of_short_sums(cuda, M, N, K):
    import torch

    q4, sc = _weights(cuda, N, K, 32, K + M)
    x = _tokens(cuda, M, K, N)
    out = torch.full((M, N), float("nan"), device=cuda)
    _gemm(out, x, q4, sc, 32)
    assert torch.equal(out, (x.double() @ _values(q4, sc, K, 32).T).float())


@pytest.mark.parametrize("M,N,K", [(12, 2601, 18971), (24, 10700, 1053), (48, 9000, 5151), (100, 5203, 1041), (300, 1701, 5153)])
def test_copied_rows(cuda, M, N, K):
    import torch

    q4, sc = _weights(cuda, N, K, 64, K)
    x = _tokens(cuda, M, K, N)
    out = torch.full((M, N), float("nan"), dtype=torch.float16, device=cuda)
    _gemm(out, x, q4, sc, 64)
    assert torch.equal(out, (x.double() @ _values(q4, sc, K, 64).T).half())


@pytest.mark.parametrize("M,N,K", [(12, 2601, 18976), (24, 10704, 1056), (48, 9000, 5184), (100, 5203, 1056), (300, 5003, 1056)])
@pytest.mark.parametrize("group", [32, 128])
def test_scales_far_apart(cuda, M, N, K, group):
    """Scales of 8 significant bits, spread over 2^20 within a row and 2^12 from row to row, tokens over 2^8.

    An fp16 output is off by half a step, 2^-11 of it (2^-25 where subnormal).  The accumulator drops, at each step of
    16 products, what of them and of the sum so far lies below 2^-24 of the largest, none of which exceeds
    sum |x w|: at most 17 * 2^-24 of that a step."""
    import torch

    g = torch.Generator(device=cuda).manual_seed(K + M)
    q4, _ = _weights(cuda, N, K, group, 3)
    ng = -(-K // group)
    sc = torch.ldexp(1 + torch.rand((N, ng), device=cuda, generator=g), torch.randint(-18, 2, (N, ng), device=cuda, generator=g))
    sc = (sc * 2.0 ** torch.randint(-12, 1, (N, 1), device=cuda, generator=g)).bfloat16()
    x = (torch.randn((M, K), device=cuda, generator=g) * 2.0 ** torch.randint(-6, 2, (M, 1), device=cuda, generator=g)).half()
    w = _values(q4, sc, K, group)
    y, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    assert y.abs().max() < 65504
    out = torch.empty((M, N), dtype=torch.float16, device=cuda)
    _gemm(out, x, q4, sc, group)
    bound = torch.maximum(2.0 ** -11 * y.abs(), torch.full_like(y, 2.0 ** -25)) + -(-K // 16) * 17 * 2.0 ** -24 * size
    assert ((out.double() - y).abs() <= bound).all()
    # one large scale a row, over codes of the value 0: the others, down to 2^-29 of it, keep all their bits
    q, s = q4.clone(), torch.full((N, ng), 2.0 ** -19, device=cuda).bfloat16()
    q[:, :group // 2] = 0x88
    s[:, 0] = 2.0 ** 10
    s[:, 1::3] *= 1.9921875  # all eight bits of a scale
    x = _tokens(cuda, M, K, N) * 64
    _gemm(out, x, q, s, group)
    y = x.double() @ _values(q, s, K, group).T
    size = x.double().abs() @ _values(q, s, K, group).abs().T
    bound = torch.maximum(2.0 ** -11 * y.abs(), torch.full_like(y, 2.0 ** -25)) + -(-K // 16) * 17 * 2.0 ** -24 * size
    assert ((out.double() - y).abs() <= bound).all()


@pytest.mark.parametrize("M,N,K", [(12, 2601, 18976), (24, 10704, 1056), (48, 10800, 1056), (100, 5203, 1056), (300, 5003, 1056),
                                   (24, 10700, 1053)])
def test_bad_tokens_stay_in_their_row(cuda, M, N, K):
    import torch

    q4, sc = _weights(cuda, N, K, 64, M)
    x = _tokens(cuda, M, K, N)
    w = _values(q4, sc, K, 64)
    y = x.double() @ w.T
    x[M // 2, 17], x[0, K - 1], x[M - 1, 40] = float("nan"), float("inf"), -float("inf")
    out = torch.full((M, N), 5.0, dtype=torch.float16, device=cuda)
    _gemm(out, x, q4, sc, 64)
    assert out[M // 2].isnan().all()
    for m, k, sign in ((0, K - 1, 1.0), (M - 1, 40, -1.0)):
        zero = w[:, k] == 0
        assert torch.equal(out[m].isnan(), zero)
        assert torch.equal(out[m][~zero].double(), sign * torch.sign(w[:, k][~zero]) * float("inf"))
    good = [m for m in range(M) if m not in (0, M // 2, M - 1)]
    assert torch.equal(out[good], y[good].half())


@pytest.mark.parametrize("bad", ["inf", "nan"])
def test_bad_scales_stay_in_their_row(cuda, bad):
    """A group of an infinite scale (quantized from an infinity) or of NaN: its row of weights gives NaN, or where
    its codes are not zero an infinity, as the formula has it, and the other rows are as they were."""
    import torch

    M, N, K, group = 40, 13000, 1056, 32
    q4, sc = _weights(cuda, N, K, group, 4)
    x = _tokens(cuda, M, K, 5)
    sc[7, 3] = sc[300, 32] = sc[N - 1, 0] = float(bad)
    q4[7, 48:64] = 0x88  # the value 0 throughout, as quantizing leaves it
    y = x.double() @ _values(q4, sc, K, group).T
    assert y[:, 7].isnan().all()
    out = torch.empty((M, N), dtype=torch.float16, device=cuda)
    _gemm(out, x, q4, sc, group)
    rows = torch.ones(N, dtype=torch.bool, device=cuda)
    rows[[7, 300, N - 1]] = False
    assert torch.equal(out[:, rows], y[:, rows].half())
    assert not out[:, ~rows].isfinite().any() and out[:, 7].isnan().all()


def test_repeats_bit_for_bit(cuda):
    """The join of a split tile's pieces has an order of its own."""
    import torch

    for M, N, K in ((12, 2601, 18944), (48, 9000, 5184), (300, 5003, 1056)):
        q4, sc = _weights(cuda, N, K, 128, M)
        x = torch.randn((M, K), device=cuda, generator=torch.Generator(device=cuda).manual_seed(M)).half()
        outs = [torch.empty((M, N), dtype=torch.float16, device=cuda) for _ in range(4)]
        for o in outs:
            _gemm(o, x, q4, sc, 128)
        assert all(torch.equal(outs[0], o) for o in outs[1:])


def _job(cuda, M, N, K, seed):
    import torch

    q4, sc = _weights(cuda, N, K, 64, seed)
    x = _tokens(cuda, M, K, seed + 1)
    want = (x.double() @ _values(q4, sc, K, 64).T).half()
    return x, q4, sc, want, torch.full((M, N), float("nan"), dtype=torch.float16, device=cuda)


# split over K with partial sums and counters; whole tiles; copied rows
JOBS = [(12, 2601, 18944), (300, 2000, 1056), (24, 10700, 1053), (64, 7000, 5184)]


def _check(jobs):
    import torch

    torch.cuda.synchronize()
    for i, (_, _, _, want, out) in enumerate(jobs):
        assert torch.equal(out, want), i
        out.fill_(float("nan"))
    torch.cuda.synchronize()


def test_graphs_of_one_stream_beside_each_other_and_beside_its_calls(cuda):
    """Captured as a stream's first calls, replayed on other streams at once beside calls on the stream."""
    import torch

    st, others = torch.cuda.Stream(), [torch.cuda.Stream() for _ in JOBS]
    for again in range(3):  # the scratch of graphs that are gone is taken again
        jobs = [_job(cuda, *j, 10 * again + i) for i, j in enumerate(JOBS)] + [_job(cuda, 33, 16000, 1056, 40 + again)]
        torch.cuda.synchronize()
        graphs = []
        for x, q4, sc, _, out in jobs[:-1]:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                _gemm(out, x, q4, sc, 64, stream=st)
                _gemm(out, x, q4, sc, 64, stream=st)
            graphs.append(g)
        for _ in range(15):
            for g, o in zip(graphs, others):
                with torch.cuda.stream(o):
                    g.replay()
            x, q4, sc, _, out = jobs[-1]
            _gemm(out, x, q4, sc, 64, stream=st)
        _check(jobs)
        del graphs, g


def test_two_branches_of_one_capture(cuda):
    import torch

    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    jobs = [_job(cuda, 64, 7000, 5184, 70), _job(cuda, 12, 2601, 18944, 71)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=a):
        b.wait_stream(a)
        for (x, q4, sc, _, out), s in zip(jobs, (a, b)):
            _gemm(out, x, q4, sc, 64, stream=s)
        a.wait_stream(b)
    for _ in range(15):
        g.replay()
    _check(jobs)


def test_streams_at_once(cuda):
    import torch

    jobs = [_job(cuda, *j, 20 + i) for i, j in enumerate(JOBS)]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(15):
        for (x, q4, sc, _, out), s in zip(jobs, streams):
            _gemm(out, x, q4, sc, 64, stream=s)
    _check(jobs)


def test_a_graph_outlives_larger_calls_on_its_stream(cuda):
    import torch

    st = torch.cuda.Stream()
    small, big = _job(cuda, 24, 10704, 1056, 1), _job(cuda, 24, 40000, 4127, 2)  # the second copies 165 MB of rows
    torch.cuda.synchronize()
    x, q4, sc, _, out = small
    _gemm(out, x, q4, sc, 64, stream=st)
    _check([small])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        _gemm(out, x, q4, sc, 64, stream=st)
    _gemm(big[4], *big[:3], 64, stream=st)
    for _ in range(3):
        with torch.cuda.stream(st):
            g.replay()
        _gemm(big[4], *big[:3], 64, stream=st)
    _check([small, big])


def test_weights_used_right_after_they_are_written(cuda):
    """quantize, then the GEMM, with nothing between, again and again into the same codes: the scales are prepared, and
    the weights loaded, only when they are there."""
    import torch

    import vvllm_b200 as v

    M, N, K = 48, 10704, 1056
    x = torch.ones((M, K), dtype=torch.float16, device=cuda)
    q4 = torch.empty((N, K // 2), dtype=torch.uint8, device=cuda)
    sc = torch.empty((N, K // 32), dtype=torch.bfloat16, device=cuda)
    ws = [torch.full((N, K), float((-2.0) ** -i), device=cuda) for i in range(6)]
    outs = [torch.empty((M, N), dtype=torch.float16, device=cuda) for _ in ws]
    for w, o in zip(ws, outs):
        v.quantize_q4(w, q4, sc, 32)
        _gemm(o, x, q4, sc, 32)
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        s = torch.tensor(2.0 ** -i / 7, dtype=torch.float64).bfloat16().double()
        assert (o == (7 * s * K * (-1) ** i).half().to(cuda)).all(), i


def test_rows_of_a_padded_batch(cuda):
    """Rows behind those given, of tokens and outputs alike, play no part and stay as they are."""
    import torch

    M, N, K = 40, 13000, 1056
    q4, sc = _weights(cuda, N, K, 64, 6)
    x = torch.full((M + 20, K), float("nan"), dtype=torch.float16, device=cuda)
    x[:M] = _tokens(cuda, M, K, 7)
    out = torch.full((M + 20, N), -5.0, dtype=torch.float16, device=cuda)
    _gemm(out[:M], x[:M], q4, sc, 64)
    assert torch.equal(out[:M], (x[:M].double() @ _values(q4, sc, K, 64).T).half()) and (out[M:] == -5).all()
