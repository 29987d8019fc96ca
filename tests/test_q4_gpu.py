"""4-bit group-quantized weights against their definition in 64 bits.

Quantization and dequantization have to match exactly.  Linear is checked twice: on integers small
enough that every product and sum is exact in fp32, where any order of summation gives the same bits
(so a wrong index, mask or rounding shows), and on the distributions of the int8 path's tests at that
path's tolerances.
"""
import numpy as np
import pytest

from tests import q4_util as u
from tests._util import TOL_F16, TOL_F32, make_bias, make_weight, make_x, rowwise_normwise_err

pytestmark = pytest.mark.gpu

EDGE = [(1, 1), (1, 2), (3, 31), (2, 32), (5, 33), (4, 64), (7, 127), (2, 128), (3, 129), (9, 200), (16, 256),
        (2, 257), (33, 896), (17, 1001), (5, 4864)]


def _scales_t(s, cuda):
    import torch

    return torch.from_numpy(u.bf16_bits(s).view(np.int16)).to(cuda).view(torch.bfloat16)


def _quantize(cuda, w, group, bf16=False, offset=0):
    """GPU quantization of a matrix that starts `offset` elements into its buffer."""
    import torch

    import vvllm_b200 as v

    N, K = w.shape
    buf = torch.zeros(N * K + offset, dtype=torch.bfloat16 if bf16 else torch.float32, device=cuda)
    buf[offset:] = torch.from_numpy(np.ascontiguousarray(w, dtype=np.float32).ravel()).to(cuda)
    q4 = torch.full((N, (K + 1) // 2), 0xA5, dtype=torch.uint8, device=cuda)
    sc = torch.full((N, -(-K // group)), -1.0, dtype=torch.bfloat16, device=cuda)
    (v.quantize_q4_bf16 if bf16 else v.quantize_q4)(buf[offset:].view(N, K), q4, sc, group)
    torch.cuda.synchronize()
    return q4, sc


def _check_quantize(cuda, w, group, bf16=False, offset=0):
    import torch

    q4, sc = _quantize(cuda, w, group, bf16, offset)
    q, s = u.quantize(w, group)
    assert np.array_equal(sc.view(torch.int16).cpu().numpy().view(np.uint16), u.bf16_bits(s))
    assert np.array_equal(q4.cpu().numpy(), u.pack(q))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", EDGE)
def test_quantize_matches_definition(cuda, N, K, group):
    _check_quantize(cuda, make_weight(N, K, 11 * N + K), group)


@pytest.mark.parametrize("offset", [1, 2, 4, 8])
@pytest.mark.parametrize("bf16", [False, True])
def test_quantize_unaligned_and_bf16(cuda, bf16, offset):
    for N, K in [(6, 256), (5, 200), (3, 1024)]:
        w = u.round_to_bf16(make_weight(N, K, 3 + K)).astype(np.float32)
        _check_quantize(cuda, w, 64, bf16, offset)


def test_quantize_edge_values(cuda):
    """Ties, zeros, subnormals, the largest values, infinities and NaN."""
    f = np.float32
    rows = [np.zeros(128, f), np.full(128, 1e-45, f), np.full(128, -3.4e38, f), np.full(128, 7.0, f)]
    ties = np.tile(np.arange(-16, 16, dtype=f) / 2, 4)  # scale 8 / 7: no ties; scale 1 below: all of them
    rows += [ties, np.where(np.arange(128) % 32 == 0, f(7.0), np.clip(ties, -6.5, 6.5)).astype(f)]
    r = np.random.default_rng(5)
    for e in (-148, -140, -134, -133, -130, -127, -126, -100, 100, 126):
        rows.append(np.ldexp(r.standard_normal(128), e).astype(f))
    for bad in (np.nan, np.inf, -np.inf):
        row = r.standard_normal(128).astype(f)
        row[[0, 37, 127]] = bad
        rows.append(row)
    rows.append(np.full(128, np.nan, f))
    w = np.stack(rows)
    for group in (32, 64, 128):
        _check_quantize(cuda, w, group)
        _check_quantize(cuda, np.tile(w, (1, 2))[:, :-3], group)
    # every quotient near a half: w = (h + d steps) * s for random 8-bit scales s
    s = (128 + r.integers(0, 128, 256)).astype(f) * f(2.0 ** -14)
    h = r.integers(-7, 7, (256, 128)).astype(f) + f(0.5)
    near = (h * s[:, None]).astype(f)
    near = np.where(r.random(near.shape) < 0.5, np.nextafter(near, f(np.inf)), np.nextafter(near, f(-np.inf)))
    near[:, 0] = 7 * s
    _check_quantize(cuda, near, 128)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("N,K", EDGE + [(40, 3584)])
def test_dequantize_rows(cuda, N, K, group, dtype):
    import torch

    import vvllm_b200 as v

    q, s = u.quantize(make_weight(N, K, 5 * N + K), group)
    want = u.values(q, s, group).astype(dtype)
    q4, sc = torch.from_numpy(u.pack(q)).to(cuda), _scales_t(s, cuda)
    out = torch.full((N, K), 7.0, dtype=getattr(torch, dtype), device=cuda)
    v.dequantize_q4(out, q4, sc, group)
    assert np.array_equal(out.cpu().numpy(), want)
    rows = np.random.default_rng(K).integers(0, N, 9).astype(np.int32)
    rows[3], rows[5], rows[6] = rows[4], -1, N  # a repeated row; indices outside
    out = torch.full((9, K), 7.0, dtype=getattr(torch, dtype), device=cuda)
    v.dequantize_q4(out, q4, sc, group, rows=torch.from_numpy(rows).to(cuda))
    got = out.cpu().numpy()
    for r, i in enumerate(rows):
        assert np.array_equal(got[r], want[i] if 0 <= i < N else np.zeros(K, dtype)), r


def _integer_case(M, N, K, group, seed):
    """Codes, scales (powers of two), tokens, bias and residual whose sums are exact in fp32: every
    partial sum is a multiple of 1/4 below 2^22."""
    r = np.random.default_rng(seed)
    q = r.integers(-8, 8, (N, K))
    s = 2.0 ** r.integers(-2, 1, (N, -(-K // group)))
    x = r.integers(-3, 4, (M, K)).astype(np.float64)
    return q, s, x, r.integers(-50, 50, N).astype(np.float64), r.integers(-50, 50, (M, N)).astype(np.float64)


def _run_linear(cuda, x, q, s, group, xdt, odt, bias=None, residual=None, in_place=False):
    import torch

    import vvllm_b200 as v

    M, N = x.shape[0], q.shape[0]
    xt = torch.from_numpy(x).to(cuda).to(getattr(torch, xdt))
    q4, sc = torch.from_numpy(u.pack(q)).to(cuda), _scales_t(s, cuda)
    bt = None if bias is None else torch.from_numpy(bias).to(cuda).float()
    rt = None if residual is None else torch.from_numpy(residual).to(cuda).to(getattr(torch, odt))
    guard = torch.full((M + 2, N), 77.0, dtype=getattr(torch, odt), device=cuda)  # a row on either side
    out = guard[1:M + 1]
    if in_place:
        out.copy_(rt)
        rt = out
    v.linear_q4_add(out, xt, q4, sc, group, bt, rt)
    torch.cuda.synchronize()
    assert (guard[0] == 77).all() and (guard[-1] == 77).all()
    assert v.kernel_error() == 0
    return out.cpu().numpy()


def _check_integers(cuda, M, N, K, group, xdt, odt, seed=0):
    q, s, x, b, res = _integer_case(M, N, K, group, seed + M + 3 * N + 5 * K)
    for bias, residual, in_place in ((None, None, False), (b, res, False), (None, res, True)):
        y = u.linear(x, q, s, group, bias, residual)
        assert np.abs(y).max() < 2 ** 22
        got = _run_linear(cuda, x, q, s, group, xdt, odt, bias, residual, in_place)
        with np.errstate(over="ignore"):
            assert np.array_equal(got, y.astype(odt)), (bias is None, in_place)


LINEAR = [(1, 1, 1), (1, 5, 31), (2, 16, 32), (3, 17, 33), (1, 16, 128), (4, 33, 96), (5, 40, 160), (8, 15, 129),
          (9, 100, 224), (1, 896, 896), (2, 1000, 1001), (7, 48, 3584), (16, 64, 512), (17, 130, 640),
          (33, 257, 1184), (1, 130, 18944)]


@pytest.mark.parametrize("xdt,odt", [("float16", "float16"), ("float16", "float32"), ("float32", "float32"),
                                     ("float32", "float16")])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", LINEAR)
def test_linear_exact_on_integers(cuda, M, N, K, group, xdt, odt):
    _check_integers(cuda, M, N, K, group, xdt, odt)


@pytest.mark.parametrize("xdt", ["float16", "float32"])
@pytest.mark.parametrize("M,N,K,group", [(1, 4864, 896, 64), (1, 896, 4864, 128), (3, 3584, 3584, 128),
                                         (8, 1000, 18944, 32), (64, 500, 3584, 64), (200, 384, 1536, 128)])
def test_linear_on_model_like_data(cuda, M, N, K, group, xdt):
    q, s = u.quantize(make_weight(N, K, N + K), group)
    x = make_x(M, K, M + K)
    if xdt == "float16":
        x = x.astype(np.float16)
    b = make_bias(N, 7)
    y = u.linear(x, q, s, group, b)
    got = _run_linear(cuda, x.astype(np.float64), q, s, group, xdt, "float32", b.astype(np.float64))
    assert rowwise_normwise_err(got, y) <= TOL_F32  # exact products and fp32 sums for either input type
    got = _run_linear(cuda, x.astype(np.float64), q, s, group, xdt, "float16", b.astype(np.float64))
    assert rowwise_normwise_err(got, y) <= TOL_F16


def test_linear_wide_ranges(cuda):
    """Scales far apart within a row and from row to row, tokens of very different size, huge and tiny
    fp32 tokens: each output row and token keeps its own relative accuracy."""
    r = np.random.default_rng(3)
    N, K, group = 70, 512, 64
    q = r.integers(-8, 8, (N, K))
    s = u.round_to_bf16(np.ldexp(1 + r.random((N, K // group)), r.integers(-6, 6, (N, K // group))))
    s *= 2.0 ** r.integers(-40, 30, (N, 1))
    for M in (1, 4, 20, 40):
        x = r.standard_normal((M, K)) * 10.0 ** r.integers(-8, 4, (M, 1))
        x32 = x.astype(np.float32).astype(np.float64)
        y = u.linear(x32, q, s, group)
        got = _run_linear(cuda, x32, q, s, group, "float32", "float32")
        size = np.abs(x32) @ np.abs(u.values(q, s, group)).T  # what the sum's rounding is relative to
        assert (np.abs(got - y) <= TOL_F32 * size).all()
        x16 = (r.standard_normal((M, K)) * 2.0 ** r.integers(-6, 8, (M, 1))).astype(np.float16).astype(np.float64)
        y = u.linear(x16, q, s, group)
        got = _run_linear(cuda, x16, q, s, group, "float16", "float32")
        size = np.abs(x16) @ np.abs(u.values(q, s, group)).T
        assert (np.abs(got - y) <= TOL_F32 * size).all()


@pytest.mark.parametrize("xdt", ["float16", "float32"])
@pytest.mark.parametrize("M", [1, 5, 24, 40])
def test_linear_bad_tokens_stay_in_their_row(cuda, M, xdt):
    """A NaN or an infinity in one token leaves the other tokens' outputs as they were."""
    q, s, x, _, _ = _integer_case(M, 50, 256, 64, 9)
    x[M // 2, 17] = np.nan
    if M > 2:
        x[0, 200] = np.inf
    y = u.linear(np.where(np.isfinite(x), x, 0), q, s, 64)
    got = _run_linear(cuda, x, q, s, 64, xdt, "float32")
    assert np.isnan(got[M // 2]).all()
    if M > 2:
        w = u.values(q, s, 64)[:, 200]
        assert np.array_equal(np.isnan(got[0]), w == 0) and np.array_equal(got[0][w != 0], np.sign(w[w != 0]) * np.inf)
    good = [m for m in range(M) if np.isfinite(x[m]).all()]
    assert np.array_equal(got[good], y[good].astype(np.float32))


@pytest.mark.parametrize("what", ["q4", "scales", "x", "out"])
def test_linear_unaligned_pointers(cuda, what):
    """Views that start off a 16-byte boundary give the same results."""
    import torch

    import vvllm_b200 as v

    for M, N, K in [(1, 64, 256), (6, 50, 512), (40, 130, 256)]:
        q, s, x, _, _ = _integer_case(M, N, K, 32, 21)
        t = {"q4": torch.from_numpy(u.pack(q)).to(cuda), "scales": _scales_t(s, cuda),
             "x": torch.from_numpy(x).to(cuda).half(), "out": torch.zeros((M, N), dtype=torch.float16, device=cuda)}
        big = torch.zeros(t[what].numel() + 1, dtype=t[what].dtype, device=cuda)
        big[1:] = t[what].reshape(-1)
        t[what] = big[1:].view(t[what].shape)
        v.linear_q4(t["out"], t["x"], t["q4"], t["scales"], 32)
        assert np.array_equal(t["out"].cpu().numpy(), u.linear(x, q, s, 32).astype(np.float16)), (M, N, K)


def test_linear_repeats_bit_for_bit(cuda):
    q, s = u.quantize(make_weight(700, 3584, 2), 128)
    for M in (1, 8, 40):
        x = make_x(M, 3584, M).astype(np.float16).astype(np.float64)
        first = _run_linear(cuda, x, q, s, 128, "float16", "float32")
        for _ in range(3):
            assert np.array_equal(first, _run_linear(cuda, x, q, s, 128, "float16", "float32"))


@pytest.mark.parametrize("M", [1, 5, 12, 40, 130, 300])
@pytest.mark.parametrize("K,group", [(896, 32), (3584, 128), (18944, 64)])
@pytest.mark.parametrize("xdt", ["float16", "float32"])
def test_fp32_outputs_are_fp32_sums(cuda, M, K, group, xdt):
    """However many tokens and however long the sums.  A sum of at most K / 32 group sums, each rounded to 2^-24
    of itself, whose errors are as good as independent: about sqrt(592) * 2^-24 * (a partial sum's mean size,
    half) < 7.3e-7 of the result's deviation; the inputs' own rounding adds 2^-22 of a chunk's largest, 4 deviations
    at most: 4 * 2^-22 / sqrt(12) < 2.8e-7."""
    import torch

    import vvllm_b200 as v

    N = 640
    g = torch.Generator(device=cuda).manual_seed(K + M)
    q4 = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=cuda, generator=g)
    sc = (0.001 + 0.01 * torch.rand((N, K // group), device=cuda, generator=g)).bfloat16()
    x = torch.randn((M, K), device=cuda, generator=g).to(getattr(torch, xdt))
    w, out = torch.empty((N, K), device=cuda), torch.empty((M, N), device=cuda)
    v.dequantize_q4(w, q4, sc, group)
    v.linear_q4(out, x, q4, sc, group)
    want = x.double() @ w.double().T
    assert float((out.double() - want).norm() / want.norm()) <= 1.1e-6


@pytest.mark.parametrize("odt", ["float16", "float32"])
@pytest.mark.parametrize("xdt", ["float16", "float32"])
@pytest.mark.parametrize("M,N,K", [(1, 77, 1001), (2, 130, 3583), (8, 33, 999), (9, 129, 801), (16, 300, 2047), (17, 65, 1030),
                                   (40, 300, 775), (130, 200, 1250), (5, 50, 18943), (100, 300, 77)])
def test_linear_rows_that_are_copied_first(cuda, M, N, K, xdt, odt):
    """K no multiple of 32, large enough to be copied into padded rows (and one that is not)."""
    _check_integers(cuda, M, N, K, 64, xdt, odt)


@pytest.mark.parametrize("what", ["q4", "x"])
@pytest.mark.parametrize("M,N,K", [(1, 100, 1024), (8, 70, 2048), (40, 300, 1024)])
def test_linear_large_unaligned_pointers(cuda, what, M, N, K):
    import torch

    import vvllm_b200 as v

    q, s, x, _, _ = _integer_case(M, N, K, 128, 5)
    t = {"q4": torch.from_numpy(u.pack(q)).to(cuda), "x": torch.from_numpy(x).to(cuda).half()}
    sc, want = _scales_t(s, cuda), u.linear(x, q, s, 128)
    for off in (1, 2, 3, 7):
        big = torch.zeros(t[what].numel() + off, dtype=t[what].dtype, device=cuda)
        big[off:] = t[what].reshape(-1)
        view, out = dict(t), torch.empty((M, N), device=cuda)
        view[what] = big[off:].view(t[what].shape)
        v.linear_q4(out, view["x"], view["q4"], sc, 128)
        assert np.array_equal(out.cpu().numpy(), want.astype(np.float32)), off


@pytest.mark.parametrize("M", [1, 12])
def test_linear_bad_tokens_stay_in_their_row_when_copied(cuda, M):
    N, K = 90, 1003
    q, s, x, _, _ = _integer_case(M + 2, N, K, 64, 8)
    x = x.copy()
    x[0, 1002], x[-1, 3] = np.inf, np.nan
    got = _run_linear(cuda, x, q, s, 64, "float16", "float32")
    with np.errstate(invalid="ignore"):
        y = u.linear(x, q, s, 64)
    assert np.array_equal(got[1:-1], y[1:-1].astype(np.float32)) and np.isnan(got[-1]).all()
    assert np.array_equal(np.isfinite(got[0]), np.isfinite(y[0]))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(7, 288), (5, 1000), (33, 40), (9, 72), (64, 1016), (300, 8), (40, 2320), (1, 3544)])
def test_quantize_rows_that_end_within_a_group(cuda, N, K, group, bf16):
    """Rows of whole octets: the last group is short, and the next row starts a new one."""
    w = make_weight(N, K, N + 5 * K)
    w[:, -1] = 3.0  # the short group's largest weight is its last
    _check_quantize(cuda, u.round_to_bf16(w).astype(np.float32) if bf16 else w, group, bf16)
