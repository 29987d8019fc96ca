"""Calls of the 4-bit operators and of the logits step at the ends of what the header allows: rows longer than a
cluster's shared memory, lists longer than 16-bit counters, addresses off every alignment, penalties of any value."""
import numpy as np
import pytest

from tests import q4_util as u

pytestmark = pytest.mark.gpu


def _values(q4, sc, K, group):
    import torch

    q = torch.stack((q4 & 15, q4 >> 4), dim=-1).flatten(1)[:, :K].double() - 8
    return q * sc.double().repeat_interleave(group, dim=1)[:, :K]


@pytest.mark.parametrize("xdt", ["float16", "float32"])
@pytest.mark.parametrize("K", [65536, 131072 + 32, 262144, 524288 + 7, 1 << 20])
@pytest.mark.parametrize("M,N", [(1, 40), (2, 17), (3, 33), (9, 20), (40, 5)])
def test_very_long_rows(cuda, M, N, K, xdt):
    """Sums of a million products, exact: multiples of 1/4 whose partial sums stay below 2^22."""
    import torch

    import vvllm_b200 as v

    g = torch.Generator(device=cuda).manual_seed(K % 1000 + M)
    q4 = torch.randint(0, 256, (N, (K + 1) // 2), dtype=torch.uint8, device=cuda, generator=g)
    if K % 2:
        q4[:, -1] = (q4[:, -1] & 15) | 0x80
    sc = (2.0 ** torch.randint(-2, 1, (N, -(-K // 128)), device=cuda, generator=g)).bfloat16()
    # steps of a random walk of at most 3 * 8 each, in 2^20 steps within 12 deviations of 5.8 * 2^10 < 2^17
    x = torch.randint(-3, 4, (M, K), device=cuda, generator=g).to(getattr(torch, xdt))
    # without a drift: the codes' mean is -1/2, of the tokens 0
    y = x.double() @ _values(q4, sc, K, 128).T
    assert y.abs().max() < 2 ** 17
    out = torch.full((M, N), float("nan"), device=cuda)
    v.linear_q4(out, x, q4, sc, 128)
    assert torch.equal(out, y.float())
    assert v.kernel_error() == 0


def _off(t, by):
    """The same values, starting `by` elements into their buffer."""
    import torch

    big = torch.zeros(t.numel() + by, dtype=t.dtype, device=t.device)
    big[by:] = t.reshape(-1)
    return big[by:].view(t.shape)


@pytest.mark.parametrize("N,K", [(5, 256), (7, 1000), (64, 896), (9, 130), (33, 4864)])
@pytest.mark.parametrize("bf16", [False, True])
def test_outputs_off_every_alignment(cuda, N, K, bf16):
    """quantize and dequantize into views that start anywhere; what lies beside them stays."""
    import torch

    import vvllm_b200 as v

    r = np.random.default_rng(N + K)
    w = u.round_to_bf16(r.standard_normal((N, K))).astype(np.float32)
    wt = torch.from_numpy(w).to(cuda)
    wt = wt.bfloat16() if bf16 else wt
    for group in (32, 128):
        q, s = u.quantize(w, group)
        kb, ng = (K + 1) // 2, -(-K // group)
        rows = r.integers(-1, N + 1, 6).astype(np.int32)
        rt = torch.from_numpy(rows).to(cuda)
        for by in (1, 2, 3, 5, 8):
            qbuf = torch.full((N * kb + by + 9,), 0xA5, dtype=torch.uint8, device=cuda)
            sbuf = torch.full((N * ng + by + 9,), -1.0, dtype=torch.bfloat16, device=cuda)
            q4, sc = qbuf[by:by + N * kb].view(N, kb), sbuf[by:by + N * ng].view(N, ng)
            (v.quantize_q4_bf16 if bf16 else v.quantize_q4)(wt, q4, sc, group)
            assert np.array_equal(q4.cpu().numpy(), u.pack(q))
            assert np.array_equal(sc.contiguous().view(torch.int16).cpu().numpy().view(np.uint16), u.bf16_bits(s))
            assert (qbuf[:by] == 0xA5).all() and (qbuf[by + N * kb:] == 0xA5).all()
            assert (sbuf[:by] == -1).all() and (sbuf[by + N * ng:] == -1).all()
            for dt in ("float32", "float16"):
                want = u.values(q, s, group).astype(dt)
                obuf = torch.full((N * K + by + 9,), 7.0, dtype=getattr(torch, dt), device=cuda)
                out = obuf[by:by + N * K].view(N, K)
                v.dequantize_q4(out, q4, sc, group)
                assert np.array_equal(out.cpu().numpy(), want)
                assert (obuf[:by] == 7).all() and (obuf[by + N * K:] == 7).all()
                out = _off(torch.full((6, K), 7.0, dtype=getattr(torch, dt), device=cuda), by)
                v.dequantize_q4(out, q4, sc, group, rows=_off(rt, by))
                got = out.cpu().numpy()
                for i, n in enumerate(rows):
                    assert np.array_equal(got[i], want[n] if 0 <= n < N else np.zeros(K, dt))


@pytest.mark.parametrize("M,N,K", [(1, 70, 1024), (2, 33, 2080), (6, 50, 1024), (12, 300, 512), (300, 1701, 5216), (9, 40, 1003)])
@pytest.mark.parametrize("what", ["scales", "out", "bias", "residual"])
def test_linear_arguments_off_every_alignment(cuda, M, N, K, what):
    import torch

    import vvllm_b200 as v

    g = torch.Generator(device=cuda).manual_seed(M)
    q4 = torch.randint(0, 256, (N, (K + 1) // 2), dtype=torch.uint8, device=cuda, generator=g)
    if K % 2:
        q4[:, -1] = (q4[:, -1] & 15) | 0x80
    t = {"scales": (2.0 ** torch.randint(-2, 1, (N, -(-K // 32)), device=cuda, generator=g)).bfloat16(),
         "bias": torch.randint(-9, 10, (N,), device=cuda, generator=g).float(),
         "residual": torch.randint(-9, 10, (M, N), device=cuda, generator=g).half(),
         "out": torch.zeros((M, N), dtype=torch.float16, device=cuda)}
    x = torch.randint(-3, 4, (M, K), device=cuda, generator=g).half()
    want = (x.double() @ _values(q4, t["scales"], K, 32).T + t["bias"].double() + t["residual"].double()).half()
    for by in (1, 2, 3, 4, 7):
        a = dict(t)
        a[what] = _off(t[what], by)
        a["out"].zero_()
        v.linear_q4_add(a["out"], x, q4, a["scales"], 32, a["bias"], a["residual"])
        assert torch.equal(a["out"], want), by


def _check_logits(cuda, c, odt="float32"):
    import torch

    import vvllm_b200 as v

    t = {k: torch.from_numpy(a).to(cuda) for k, a in c.items()}
    x = t.pop("x")
    out = torch.full(x.shape, 55.0, dtype=getattr(torch, odt), device=cuda)
    tok = torch.full((x.shape[0],), -77, dtype=torch.int32, device=cuda)
    v.process_logits(out, x, tok, **t)
    want, wtok = u.logits(**c, out_dtype=np.dtype(odt))
    assert np.array_equal(out.cpu().numpy(), want, equal_nan=True)
    assert np.array_equal(tok.cpu().numpy(), wtok)


@pytest.mark.parametrize("V,hist,biases", [(5000, 40000, 0), (5000, 32767, 65534), (5000, 32768, 65535), (33, 70000, 70000),
                                           (152064, 33000, 300), (400_003, 50000, 70000)])
def test_lists_longer_than_small_counters(cuda, V, hist, biases):
    """Counts and entries of 16 and of 32 bits, on either side of the change; one token in most places of a row."""
    r = np.random.default_rng(V + hist)
    c = {"x": (4 * r.standard_normal((2, V))).astype(np.float32),
         "history": r.integers(0, V, (2, hist)).astype(np.int32), "history_len": np.array([hist, hist - 1], np.int32),
         "prompt_len": np.array([0, hist // 3], np.int32), "repetition": np.array([1.3, 0.9], np.float32),
         "presence": np.array([0.5, -0.5], np.float32), "frequency": np.array([0.001, 0.01], np.float32)}
    c["history"][0, :] = np.where(r.random(hist) < 0.99, V // 2, c["history"][0])
    c["history"][1, :] = V - 1  # every count a 16-bit slot can hold, and its top bit
    if biases:
        c["bias_ids"] = r.integers(0, V, (2, biases)).astype(np.int32)
        c["bias_ids"][0, :] = V // 2  # the last of them all
        c["bias_values"] = r.standard_normal((2, biases)).astype(np.float32)
    _check_logits(cuda, c)


@pytest.mark.parametrize("odt", ["float32", "float16"])
def test_penalties_of_any_value(cuda, odt):
    """Zero, negative, infinite and NaN penalties, biases and logits in every combination."""
    vals = np.array([0.0, -0.0, 1.0, -1.0, 2.5, -0.3, 1e-40, 3e38, -3e38, np.inf, -np.inf, np.nan], np.float32)
    rows = [(a, b, c) for a in vals for b in vals[[0, 2, 3, 9, 10, 11]] for c in vals[[0, 3, 7, 9, 11]]]
    M, V = len(rows), 4 * len(vals) + 5
    x = np.zeros((M, V), np.float32)
    x[:, :4 * len(vals)] = np.tile(vals, 4)
    history = np.tile(np.arange(2 * len(vals), dtype=np.int32), (M, 1))  # once in the prompt, or once made
    history = np.concatenate([history, np.arange(3 * len(vals) // 2, 2 * len(vals), dtype=np.int32)[None].repeat(M, 0)], axis=1)
    c = {"x": x, "history": history, "history_len": np.full(M, history.shape[1], np.int32),
         "prompt_len": np.full(M, len(vals), np.int32),
         "repetition": np.array([a for a, _, _ in rows], np.float32), "presence": np.array([b for _, b, _ in rows], np.float32),
         "frequency": np.array([f for _, _, f in rows], np.float32),
         "bias_ids": np.arange(V, dtype=np.int32)[::2].copy(), "bias_values": np.resize(vals, (V + 1) // 2).astype(np.float32),
         "allowed": np.array([[-1, 0x7FFFFFFE]], np.int32)}
    _check_logits(cuda, c, odt)


def test_rules_and_outputs_that_are_one_buffer_apart(cuda):
    """Tokens written to the column of the history that the next step reads: the call itself must be told where the
    history ends, or refuse."""
    import torch

    import vvllm_b200 as v

    hist = torch.zeros((1, 8), dtype=torch.int32, device=cuda)
    n = torch.ones(1, dtype=torch.int32, device=cuda)
    lg = torch.randn((1, 100), device=cuda)
    with pytest.raises(v.B200Q8Error, match="overlaps an input"):
        v.process_logits(None, lg, hist[0, 3:4], history=hist, history_len=n)
    v.process_logits(None, lg, hist[0, 3:4], history=hist[:, :3], history_len=n)
    assert int(hist[0, 3]) == int(lg.argmax())
