"""Several host threads calling at once: on one stream, where the launches of one call have to stay together
(they meet in the stream's scratch), and on the per-thread stream, one handle for a stream of every thread."""
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

PER_THREAD = 2  # the value of cudaStreamPerThread


def _q4_job(cuda, M, N, K, odt, seed):
    """A linear_q4 call whose sums are exact, and its result from a product in 64 bits."""
    import torch

    import vvllm_b200 as v

    g = torch.Generator(device=cuda).manual_seed(seed)
    q4 = torch.randint(0, 256, (N, (K + 1) // 2), dtype=torch.uint8, device=cuda, generator=g)
    if K % 2:
        q4[:, -1] = (q4[:, -1] & 15) | 0x80
    sc = (2.0 ** torch.randint(-2, 1, (N, -(-K // 64)), device=cuda, generator=g)).bfloat16()
    x = torch.randint(-3, 4, (M, K), device=cuda, generator=g).half()
    q = torch.stack((q4 & 15, q4 >> 4), dim=-1).flatten(1)[:, :K].double() - 8
    want = (x.double() @ (q * sc.double().repeat_interleave(64, dim=1)[:, :K]).T).to(odt)

    def call(out, stream):
        v.linear_q4(out, x, q4, sc, 64, stream=stream)

    return call, want


def _q8_job(cuda, what, seed):
    """A call of the int8 path that is several launches, and its result from one thread."""
    import torch

    import vvllm_b200 as v

    M, N, K = {"norm": (40, 3000, 1024), "silu": (40, 3000, 1024), "digits": (8, 16400, 1024), "fp32": (50, 700, 1024),
               "noalloc": (2, 40000, 1024)}[what]
    g = torch.Generator(device=cuda).manual_seed(seed)
    w = torch.randint(-127, 128, (N, K), dtype=torch.int8, device=cuda, generator=g)
    s = 0.01 + 0.01 * torch.rand(N, device=cuda, generator=g)
    x = torch.randn((M, 2 * K if what == "silu" else K), device=cuda, generator=g)
    x = x if what == "fp32" else x.half()
    norm = 1 + torch.rand(K, device=cuda, generator=g)

    def call(out, stream):
        if what == "norm":
            v.rms_norm_linear_q8(out, x, norm, 1e-6, w, s, stream=stream)
        elif what == "silu":
            v.silu_mul_linear_q8_add(out, x, w, s, stream=stream)
        elif what == "noalloc":
            st = v.lib().b200q8_linear_q8_noalloc(out.data_ptr(), 1, x.data_ptr(), 1, w.data_ptr(), s.data_ptr(), None, None,
                                                  M, N, K, stream)
            assert st == 0, v.lib().b200q8_last_error()
        else:
            v.linear_q8(out, x, w, s, stream=stream)

    want = torch.empty((M, N), dtype=torch.float32 if what == "fp32" else torch.float16, device=cuda)
    call(want, None)
    torch.cuda.synchronize()
    return call, want


def _together(cuda, jobs, streams, rounds=25):
    """Every job from a thread of its own, `rounds` times into outputs of their own, all at once."""
    import torch

    outs = [[torch.full_like(want, float("nan")) for _ in range(rounds)] for _, want in jobs]
    torch.cuda.synchronize()
    gate, errors = threading.Barrier(len(jobs)), []

    def work(i):
        try:
            gate.wait()
            for out in outs[i]:
                jobs[i][0](out, streams[i])
        except BaseException as e:  # noqa: BLE001 -- reported by the test
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    import vvllm_b200 as v

    assert v.kernel_error() == 0
    for i, (_, want) in enumerate(jobs):
        for r, out in enumerate(outs[i]):
            assert torch.equal(out, want), (i, r)


# GEMM; copied rows to the streaming kernel; copied rows to the GEMM
Q4 = {"gemm": (24, 10700, 1056, "float16"), "copied": (1, 600, 2045, "float32"), "both": (24, 10700, 1053, "float16")}


def _q4_jobs(cuda, kinds):
    import torch

    return [_q4_job(cuda, *Q4[k][:3], getattr(torch, Q4[k][3]), 100 + i) for i, k in enumerate(kinds)]


def _stream(which):
    import torch

    return {"legacy": lambda: None, "own": lambda: torch.cuda.Stream(), "per-thread": lambda: PER_THREAD}[which]()


@pytest.mark.parametrize("which", ["legacy", "own", "per-thread"])
@pytest.mark.parametrize("kinds", [("gemm", "gemm"), ("copied", "copied"), ("both", "both"), ("gemm", "copied", "both")],
                         ids="-".join)
def test_q4_calls_from_several_threads(cuda, kinds, which):
    jobs = _q4_jobs(cuda, kinds)
    s = _stream(which)
    _together(cuda, jobs, [s] * len(jobs))


@pytest.mark.parametrize("which", ["legacy", "own", "per-thread"])
@pytest.mark.parametrize("what", ["norm", "silu", "digits", "fp32"])
def test_q8_calls_from_several_threads(cuda, what, which):
    s = _stream(which)
    _together(cuda, [_q8_job(cuda, what, 7 + i) for i in range(2)], [s] * 2)


@pytest.mark.parametrize("which", ["legacy", "own"])
def test_noalloc_calls_from_several_threads_of_one_stream(cuda, which):
    s = _stream(which)
    handle = None if s is None else s.cuda_stream
    _together(cuda, [_q8_job(cuda, "noalloc", 17 + i) for i in range(2)], [handle] * 2)


def test_threads_that_capture_and_call(cuda):
    """One thread captures graphs on a stream of its own and replays them while another calls on its stream."""
    import torch

    jobs = _q4_jobs(cuda, ("gemm", "both"))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [torch.full_like(want, float("nan")) for _, want in jobs]
    torch.cuda.synchronize()
    for (call, _), out, st in zip(jobs, outs, streams):  # scratch of either stream: allocated before any capture
        call(out, st)
    torch.cuda.synchronize()
    errors = []

    def capture():
        try:
            for _ in range(5):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=streams[0], capture_error_mode="thread_local"):
                    jobs[0][0](outs[0], streams[0])
                with torch.cuda.stream(streams[0]):
                    for _ in range(5):
                        g.replay()
                streams[0].synchronize()
        except BaseException as e:  # noqa: BLE001 -- reported by the test
            errors.append(e)

    t = threading.Thread(target=capture)
    t.start()
    for _ in range(60):
        jobs[1][0](outs[1], streams[1])
    t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for (_, want), out in zip(jobs, outs):
        assert np.array_equal(out.cpu().numpy(), want.cpu().numpy())


FIRST_CALLS = """
import threading
import torch
import vvllm_b200 as v

x, q4 = torch.ones((24, 64), device="cuda").half(), torch.full((300, 32), 0x99, dtype=torch.uint8, device="cuda")
sc = torch.ones((300, 1), dtype=torch.bfloat16, device="cuda")
outs = [torch.zeros((24, 300), device="cuda") for _ in range(16)]
torch.cuda.synchronize()
v.lib()
gate = threading.Barrier(16)

def work(o):
    gate.wait()
    v.linear_q4(o, x, q4, sc, 64)

threads = [threading.Thread(target=work, args=(o,)) for o in outs]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
assert all((o == 64).all() for o in outs)
print("ok")
"""


def test_the_first_calls_of_a_process_at_once(cuda):
    """What the library looks up once a process is looked up by sixteen threads together."""
    import subprocess
    import sys

    from tests.conftest import ROOT

    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
