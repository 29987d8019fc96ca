"""Device memory that calls with scratch hold: what the largest call so far needed, not twice that, nor the buffers it
outgrew, unless a captured graph may still use them; and what a graph held can be had again when it is gone."""
import time

import pytest

pytestmark = pytest.mark.gpu

MB = 1 << 20


def _job(cuda, N, K, M=1):
    """A call whose rows are copied first: N * K / 2 bytes of scratch, about."""
    import torch

    q4 = torch.full((N, (K + 1) // 2), 0x99, dtype=torch.uint8, device=cuda)  # ones
    q4[:, -1] = 0x89
    return (torch.empty((M, N), device=cuda), torch.ones((M, K), dtype=torch.float16, device=cuda), q4,
            torch.ones((N, -(-K // 128)), dtype=torch.bfloat16, device=cuda), 128)


def _used(torch):
    torch.cuda.synchronize()
    free, total = torch.cuda.mem_get_info()
    return (total - free) / MB


def _call(job, stream):
    import torch

    import vvllm_b200 as v

    job[0].zero_()
    torch.cuda.synchronize()
    v.linear_q4(*job, stream=stream)


def _right(job):
    import torch

    torch.cuda.synchronize()
    assert (job[0] == job[1].shape[1]).all()


def test_a_call_that_needs_a_little_more(cuda):
    import torch

    jobs = [_job(cuda, 60000, k) for k in (8191, 8223, 8255, 8287)]  # 246 MB of copied rows and 1 MB more each time
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    before = _used(torch)
    for job in jobs:
        _call(job, stream)
        _right(job)
        held = _used(torch) - before
        assert held < 60000 * 4144 / MB + 64, f"{held:.0f} MB"  # 237 MB, and partial sums and counters of their own


def test_small_needs_are_met_in_few_steps(cuda):
    """Below 64 MB sizes double: forty sizes, each a little larger, do not make forty allocations that wait for the GPU."""
    import torch

    jobs = [_job(cuda, 2000, 2047 + 64 * i) for i in range(40)]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    seen = set()
    for job in jobs:
        _call(job, stream)
        _right(job)
        seen.add(round(_used(torch)))
    assert len(seen) <= 5, seen


def test_what_an_int8_graph_holds_stays(cuda):
    """The int8 calls of a captured graph use the stream's scratch: a larger call later must not free it."""
    import torch

    import vvllm_b200 as v

    stream = torch.cuda.Stream()
    g = torch.Generator(device=cuda).manual_seed(0)
    w = torch.randint(-8, 8, (3000, 1024), dtype=torch.int8, device=cuda, generator=g)
    s, norm = torch.ones(3000, device=cuda), torch.ones(1024, device=cuda)
    x = torch.randn((40, 1024), device=cuda, generator=g).half()
    out, want = (torch.empty((40, 3000), dtype=torch.float16, device=cuda) for _ in range(2))
    torch.cuda.synchronize()
    v.rms_norm_linear_q8(want, x, norm, 1e-6, w, s, stream=stream)  # writes the normed tokens into the scratch
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        v.rms_norm_linear_q8(out, x, norm, 1e-6, w, s, stream=stream)
    big = _job(cuda, 60000, 8191)
    _call(big, stream)  # the scratch grows
    _right(big)
    junk = [torch.full((MB,), float("nan"), device=cuda) for _ in range(8)]  # into what might have been freed
    for _ in range(3):
        with torch.cuda.stream(stream):
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert len(junk) == 8


def test_a_graph_holds_what_it_needs_and_gives_it_back(cuda):
    import torch

    import vvllm_b200 as v

    stream = torch.cuda.Stream()
    large, small = _job(cuda, 60000, 4607), _job(cuda, 3000, 2047)  # 138 MB and 3 MB
    torch.cuda.synchronize()

    def capture(job):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            v.linear_q4(*job, stream=stream)
        with torch.cuda.stream(stream):
            job[0].zero_()
            g.replay()
        _right(job)
        return g

    torch.cuda.empty_cache()
    start = _used(torch)
    g1 = capture(large)
    held = _used(torch) - start
    assert held < 60000 * 2304 / MB + 32, f"{held:.0f} MB"  # 132 MB: not rounded up to 256
    g2 = capture(large)
    assert _used(torch) - start < 2 * (60000 * 2304 / MB + 32)
    del g1, g2
    for _ in range(100):  # the graphs' end is told from another thread: a while later a capture frees what it cannot use
        g3 = capture(small)
        now = _used(torch) - start
        if now < 32:
            break
        del g3
        time.sleep(0.05)
    assert now < 32, f"{now:.0f} MB still held"


def test_captures_in_turn_do_not_pile_up(cuda):
    import torch

    import vvllm_b200 as v

    stream = torch.cuda.Stream()
    jobs = [_job(cuda, n, 2047, m) for n, m in ((3000, 1), (20000, 1), (60000, 1), (9000, 4))]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    start = _used(torch)
    for i in range(24):
        job = jobs[i % 4]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            v.linear_q4(*job, stream=stream)
        with torch.cuda.stream(stream):
            job[0].zero_()
            g.replay()
        _right(job)
        del g
        time.sleep(0.01)
    held = _used(torch) - start
    assert held < 4 * 64 + 64, f"{held:.0f} MB"
