"""A host thread's first CUDA call of any kind is a call of this library: no context is bound to the thread yet."""
import threading

import pytest

pytestmark = pytest.mark.gpu


def _in_a_new_thread(f):
    errors = []

    def run():
        try:
            f()
        except BaseException as e:  # noqa: BLE001 -- reported by the test
            errors.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    assert not errors, errors


@pytest.mark.parametrize("M,N,K,dtype", [(1, 600, 1024, "float16"), (2, 600, 1024, "float32"), (8, 600, 1024, "float16"),
                                         (24, 10700, 1056, "float16"), (1, 600, 1021, "float16")])
def test_linear_q4(cuda, M, N, K, dtype):
    import torch

    import vvllm_b200 as v

    g = torch.Generator(device=cuda).manual_seed(M)
    q4 = torch.randint(0, 256, (N, (K + 1) // 2), dtype=torch.uint8, device=cuda, generator=g)
    sc = (2.0 ** torch.randint(-2, 1, (N, -(-K // 64)), device=cuda, generator=g)).bfloat16()
    x = torch.randint(-3, 4, (M, K), device=cuda, generator=g).to(getattr(torch, dtype))
    out = torch.full((M, N), float("nan"), dtype=torch.float16, device=cuda)
    torch.cuda.synchronize()
    _in_a_new_thread(lambda: v.linear_q4(out, x, q4, sc, 64))
    torch.cuda.synchronize()
    q = torch.stack((q4 & 15, q4 >> 4), dim=-1).flatten(1)[:, :K].double() - 8
    want = x.double() @ (q * sc.double().repeat_interleave(64, dim=1)[:, :K]).T
    assert torch.equal(out, want.half())


@pytest.mark.parametrize("M,N,K,dtype", [(1, 60000, 1024, "float16"), (8, 20000, 1024, "float16"), (40, 600, 1024, "float16"),
                                         (6, 600, 1024, "float32")])
def test_linear_q8(cuda, M, N, K, dtype):
    import torch

    import vvllm_b200 as v

    g = torch.Generator(device=cuda).manual_seed(M)
    w = torch.randint(-8, 8, (N, K), dtype=torch.int8, device=cuda, generator=g)
    s = torch.ones(N, device=cuda)
    x = torch.randint(-3, 4, (M, K), device=cuda, generator=g).to(getattr(torch, dtype))
    out = torch.full((M, N), float("nan"), dtype=torch.float16, device=cuda)
    torch.cuda.synchronize()
    _in_a_new_thread(lambda: v.linear_q8(out, x, w, s))
    torch.cuda.synchronize()
    assert torch.equal(out, (x.double() @ w.double().T).half())


def test_rows_and_logits(cuda):
    import torch

    import vvllm_b200 as v

    w = torch.randn((64, 256), device=cuda)
    q4, sc = torch.empty((64, 128), dtype=torch.uint8, device=cuda), torch.empty((64, 4), dtype=torch.bfloat16, device=cuda)
    vals, tok = torch.empty_like(w), torch.empty(64, dtype=torch.int32, device=cuda)
    torch.cuda.synchronize()
    _in_a_new_thread(lambda: v.quantize_q4(w, q4, sc, 64))
    _in_a_new_thread(lambda: v.dequantize_q4(vals, q4, sc, 64))
    _in_a_new_thread(lambda: v.process_logits(None, w, tok))
    torch.cuda.synchronize()
    # half a step of the codes, and half a bf16 step of the scale at the outermost
    assert ((vals - w).abs() <= sc.float().repeat_interleave(64, dim=1) * (0.5 + 8 * 2.0 ** -8)).all()
    assert torch.equal(tok.long(), w.argmax(dim=1))
