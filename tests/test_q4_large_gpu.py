"""Offsets behind 32 bits: outputs, inputs and weights of more than 2^31 elements."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _rows(at, last):
    """Rows to look at: the first, `at` (behind element 2^31), the middle and the last."""
    return [0, 1, at, last // 2, last - 1, last]


@pytest.fixture
def room(cuda):
    import torch

    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def test_a_linear_of_more_than_2_31_outputs(cuda, room):
    import torch

    import vvllm_b200 as v

    M, N, K = 17001, 152064, 128  # 2.6e9 fp16
    r = torch.Generator(device=cuda).manual_seed(0)
    q4 = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=cuda, generator=r)
    sc = torch.full((N, 2), 0.25, dtype=torch.bfloat16, device=cuda)
    x = torch.randint(-3, 4, (M, K), device=cuda, generator=r).half()
    out = torch.empty((M, N), dtype=torch.float16, device=cuda)
    v.linear_q4(out, x, q4, sc, 64)
    w = torch.empty((N, K), device=cuda)
    v.dequantize_q4(w, q4, sc, 64)
    at = _rows((1 << 31) // N + 1, M - 1)
    # sums of multiples of a quarter, |sum| <= 128 * 3 * 2: exact in fp32, then rounded once to fp16
    want = x[at].double() @ w.double().T
    got = out[at].double()
    assert ((got - want).abs() <= want.abs() * 2.0 ** -11).all()


def test_a_lookup_of_more_than_2_31_values(cuda, room):
    import torch

    import vvllm_b200 as v

    R, N, K = 600011, 5000, 3584
    r = torch.Generator(device=cuda).manual_seed(1)
    q4 = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=cuda, generator=r)
    sc = torch.full((N, K // 128), 2.0, dtype=torch.bfloat16, device=cuda)
    rows = torch.randint(0, N, (R,), dtype=torch.int32, device=cuda, generator=r)
    out = torch.empty((R, K), dtype=torch.float16, device=cuda)
    v.dequantize_q4(out, q4, sc, 128, rows=rows)
    at = torch.tensor(_rows((1 << 31) // K + 1, R - 1), device=cuda)
    c = q4[rows[at].long()].int()
    want = (torch.stack([c & 15, c >> 4], dim=-1).reshape(len(at), K) - 8) * 2
    assert torch.equal(out[at].int(), want)


@pytest.mark.parametrize("K", [4096, 4097])
def test_weights_of_more_than_2_31_values(cuda, room, K):
    """Quantized, read back and multiplied by a token."""
    import torch

    import vvllm_b200 as v

    N = 540007  # 2.2e9 weights: 1.1 GB of codes
    w = torch.empty((N, K), dtype=torch.bfloat16, device=cuda)
    row = (torch.arange(K, device=cuda) % 15 - 7).to(torch.bfloat16)
    mult = 2.0 ** (torch.arange(N, device=cuda) % 5)
    torch.mul(row[None, :], mult[:, None].to(torch.bfloat16), out=w)
    q4 = torch.empty((N, (K + 1) // 2), dtype=torch.uint8, device=cuda)
    sc = torch.empty((N, -(-K // 64)), dtype=torch.bfloat16, device=cuda)
    v.quantize_q4_bf16(w, q4, sc, 64)
    at = _rows((1 << 31) // K + 1, N - 1)
    back = torch.empty((N, K), dtype=torch.float16, device=cuda)
    v.dequantize_q4(back, q4, sc, 64)
    # every whole group's largest weight is 7 times a power of two, which becomes its scale: all exact
    whole = K // 64 * 64
    assert torch.equal(back[at][:, :whole].double(), w[at][:, :whole].double())
    x = torch.ones((1, K), device=cuda)
    x[0, whole:] = 0
    out = torch.empty((1, N), device=cuda)
    v.linear_q4(out, x, q4, sc, 64)
    want = mult.double() * row[:whole].double().sum()
    assert torch.equal(out[0].double(), want)


def test_logits_of_more_than_2_31_elements(cuda, room):
    import torch

    import vvllm_b200 as v

    M, V = 14501, 152065
    lg = torch.zeros((M, V), dtype=torch.float16, device=cuda)
    best = torch.arange(M, device=cuda) * 7919 % V
    lg[torch.arange(M, device=cuda), best] = 5.0
    hist = torch.stack([best, (best + 1) % V], dim=1).int()
    tok = torch.empty(M, dtype=torch.int32, device=cuda)
    v.process_logits(lg, lg, tok, history=hist, history_len=torch.full((M,), 2, dtype=torch.int32, device=cuda),
                     presence=torch.full((M,), 1.0, device=cuda))
    assert np.array_equal(tok.cpu().numpy(), best.cpu().numpy())
    for m in _rows((1 << 31) // V + 1, M - 1):
        row, b = lg[m], int(best[m])
        assert row[b] == 4 and row[(b + 1) % V] == -1 and int((row != 0).sum()) == 2
