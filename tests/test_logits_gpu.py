"""process_logits against the rules restated token by token: outputs and tokens match exactly (each
operation is one fp32 rounding on either side)."""
import numpy as np
import pytest

from tests import q4_util as u

pytestmark = pytest.mark.gpu


def _case(M, V, hist, biases, mask, seed, xdt="float32"):
    r = np.random.default_rng(seed)
    c = {"x": (4 * r.standard_normal((M, V))).astype(xdt)}
    if hist:
        c["history"] = (V * r.random((M, hist)) ** 3).astype(np.int32)
        c["history_len"] = r.integers(0, hist + 1, M).astype(np.int32)
        c["prompt_len"] = (c["history_len"] // 2).astype(np.int32)
        c["repetition"] = (0.8 + r.random(M)).astype(np.float32)
        c["presence"] = r.standard_normal(M).astype(np.float32)
        c["frequency"] = r.standard_normal(M).astype(np.float32)
    if biases:
        c["bias_ids"] = r.integers(0, V, (M, biases)).astype(np.int32)
        c["bias_values"] = (3 * r.standard_normal((M, biases))).astype(np.float32)
        c["bias_len"] = r.integers(0, biases + 1, M).astype(np.int32)
    if mask:
        c["allowed"] = r.integers(-2**31, 2**31, (M, (V + 31) // 32)).astype(np.int32)
    return c


def _run(cuda, c, odt="float32", out=None, token=True, stream=None):
    import torch

    import vvllm_b200 as v

    t = {k: torch.from_numpy(a).to(cuda) for k, a in c.items()}
    x = t.pop("x")
    M, V = x.shape
    if out is None:
        out = torch.full((M, V), 55.0, dtype=getattr(torch, odt), device=cuda)
    am = torch.full((M,), -77, dtype=torch.int32, device=cuda) if token else None
    v.process_logits(out, x, am, **t, stream=stream)
    torch.cuda.synchronize()
    return out.cpu().numpy(), am.cpu().numpy() if token else None


def _check(cuda, c, odt="float32"):
    out, tok = _run(cuda, c, odt)
    want, wtok = u.logits(**c, out_dtype=np.dtype(odt))
    assert np.array_equal(out, want, equal_nan=True)
    assert np.array_equal(tok, wtok)


@pytest.mark.parametrize("xdt,odt", [("float32", "float32"), ("float16", "float16"), ("float16", "float32"),
                                     ("float32", "float16")])
@pytest.mark.parametrize("M,V,hist,biases,mask", [
    (1, 1, 1, 1, True), (2, 31, 5, 0, True), (1, 32, 0, 3, False), (3, 33, 40, 7, True), (5, 257, 0, 0, True),
    (2, 1000, 300, 20, False), (7, 4099, 1000, 300, True), (1, 32001, 2000, 0, False), (3, 50257, 100, 50, True),
    (1, 151936, 5000, 0, True)])
def test_matches_rules(cuda, M, V, hist, biases, mask, xdt, odt):
    _check(cuda, _case(M, V, hist, biases, mask, M + V, xdt), odt)


def test_vocabulary_beyond_one_pass_of_counters(cuda):
    """More tokens than the counters of one cluster hold: the slices are passed in turns."""
    c = _case(2, 700_001, 3000, 100, True, 4)
    c["history"][:, ::3] = np.random.default_rng(1).integers(500_000, 700_001, c["history"][:, ::3].shape)
    c["history_len"][:] = 3000
    _check(cuda, c)


def test_many_rows(cuda):
    _check(cuda, _case(300, 700, 64, 10, True, 8))


def test_rules_one_by_one(cuda):
    full = _case(4, 3001, 500, 60, True, 17)
    x = {"x": full["x"]}
    hist = {k: full[k] for k in ("x", "history", "history_len")}
    _check(cuda, x)
    _check(cuda, hist)
    for k in ("repetition", "presence", "frequency"):
        _check(cuda, {**hist, k: full[k]})
        _check(cuda, {**hist, k: full[k], "prompt_len": full["prompt_len"]})
    _check(cuda, {**x, "bias_ids": full["bias_ids"], "bias_values": full["bias_values"]})
    _check(cuda, {**x, "allowed": full["allowed"]})
    # penalties without a history have nothing to act on
    _check(cuda, {**x, "allowed": full["allowed"][:1]})  # one mask for all rows
    import torch

    out, _ = _run(cuda, {**x, "repetition": full["repetition"]})
    assert np.array_equal(out, full["x"])
    assert torch.cuda.is_available()


def test_rows_shared_by_all(cuda):
    c = _case(5, 999, 80, 30, True, 23)
    for k in ("history", "bias_ids", "bias_values", "allowed"):
        c[k] = c[k][0]
    _check(cuda, c)


def test_ids_and_lengths_outside_are_ignored(cuda):
    c = _case(3, 500, 64, 16, False, 5)
    c["history"][:, ::4] = [-1] * 16
    c["history"][:, 1::8] = 500
    c["history"][:, 2::8] = 2**31 - 1
    c["bias_ids"][:, ::3] = -2**31
    c["history_len"][:] = [-5, 1000, 64]
    c["prompt_len"][:] = [3, -1, 2000]
    c["bias_len"][:] = [-1, 999, 16]
    _check(cuda, c)


def test_masks_leave_nothing_or_little(cuda):
    c = _case(6, 1003, 50, 8, True, 31)
    c["allowed"][:] = 0
    c["allowed"][1, 0] = 1          # only token 0
    c["allowed"][2, 31] = 1 << 10   # only token 1002, the last
    c["allowed"][3, 31] = -1 << 11  # only bits behind the vocabulary
    c["allowed"][4, 5] = -2**31     # only token 191, whose logit is -inf
    c["x"][4] = np.nan
    c["x"][4, 191] = -np.inf
    c["x"][5] = np.inf              # nothing allowed at all
    _check(cuda, c)
    _, tok = _run(cuda, c)
    assert tok.tolist() == [-1, 0, 1002, -1, 191, -1]


def test_nan_infinity_and_ties(cuda):
    x = np.zeros((8, 300), np.float32)
    x[0] = np.nan
    x[1, 0] = np.nan
    x[2, 5] = np.nan
    x[2, 7] = 1
    x[3] = -np.inf
    x[4, 100] = x[4, 200] = np.inf
    x[5, ::2] = -0.0  # -0 and 0 are equal: the first wins
    x[6] = -1
    x[6, 250] = x[6, 30] = -0.5
    x[7, 10] = x[7, 20] = 65519.0  # equal once stored as fp16
    x[7, 20] = 65504.0
    for odt in ("float32", "float16"):
        _check(cuda, {"x": x}, odt)
    _check(cuda, {"x": x, "allowed": np.full((8, 10), -2, np.int32)})  # without token 0 and each 32nd


def test_repetition_of_zero_and_signs(cuda):
    c = {"x": np.tile(np.array([[2.0, -2.0, 0.0, -0.0, np.inf, -np.inf, np.nan, 1.0]], np.float32), (4, 1)),
         "history": np.tile(np.arange(7, dtype=np.int32), (4, 1)), "history_len": np.full(4, 7, np.int32),
         "repetition": np.array([0.0, 1.5, 1e38, np.inf], np.float32)}
    _check(cuda, c)


@pytest.mark.parametrize("xdt", ["float32", "float16"])
def test_strides_in_place_and_no_output(cuda, xdt):
    import torch

    import vvllm_b200 as v

    c = _case(5, 777, 50, 10, True, 2, xdt)
    want, wtok = u.logits(**c, out_dtype=np.dtype(xdt))
    t = {k: torch.from_numpy(a).to(cuda) for k, a in c.items()}
    x = t.pop("x")
    for pad in (3, 7, 23):  # row strides off and on 16-byte boundaries; what lies behind the rows stays
        big = torch.full((5, 777 + pad), 9.0, dtype=x.dtype, device=cuda)
        big[:, :777] = x
        wide = {k: torch.nn.functional.pad(a, (0, 2)) if a.dim() == 2 else a for k, a in t.items()}
        wide = {k: a[:, :-2] if a.dim() == 2 else a for k, a in wide.items()}
        am = torch.empty(5, dtype=torch.int32, device=cuda)
        v.process_logits(None, big[:, :777], am, **wide)
        assert np.array_equal(am.cpu().numpy(), wtok) and torch.equal(big[:, :777], x)
        v.process_logits(big[:, :777], big[:, :777], None, **wide)
        assert np.array_equal(big[:, :777].cpu().numpy(), want) and (big[:, 777:] == 9).all()


def test_single_rows_of_any_start(cuda):
    """One row at every element offset: the vector path's edges."""
    import torch

    import vvllm_b200 as v

    for dt in ("float32", "float16"):
        c = _case(1, 1500, 30, 5, True, 77, dt)
        want, wtok = u.logits(**c, out_dtype=np.dtype(dt))
        t = {k: torch.from_numpy(a).to(cuda) for k, a in c.items()}
        x = t.pop("x")
        for i in range(9):
            for o in range(0, 9, 3):
                src = torch.zeros(1520, dtype=x.dtype, device=cuda)
                dst = torch.full((1520,), 3.0, dtype=x.dtype, device=cuda)
                src[i:i + 1500] = x[0]
                am = torch.empty(1, dtype=torch.int32, device=cuda)
                v.process_logits(dst[o:o + 1500].view(1, -1), src[i:i + 1500].view(1, -1), am, **t)
                got = dst.cpu().numpy()
                assert np.array_equal(got[o:o + 1500], want[0]) and am.item() == wtok[0]
                assert (got[:o] == 3).all() and (got[o + 1500:] == 3).all()
