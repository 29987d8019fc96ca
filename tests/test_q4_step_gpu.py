"""The 4-bit operators and the logits step together, as a decode loop uses them, and the ways a program may
call them: from a captured graph, on other streams at once, on padded batches and in place."""
import numpy as np
import pytest

from tests import q4_util as u
from tests._util import make_weight, rowwise_normwise_err

pytestmark = pytest.mark.gpu


def _quantized(cuda, w, group):
    import torch

    import vvllm_b200 as v

    N, K = w.shape
    wt = torch.from_numpy(w).to(cuda)
    q4 = torch.empty((N, (K + 1) // 2), dtype=torch.uint8, device=cuda)
    sc = torch.empty((N, -(-K // group)), dtype=torch.bfloat16, device=cuda)
    v.quantize_q4(wt, q4, sc, group)
    return q4, sc


def _host_values(q4, sc, K, group):
    c = q4.cpu().numpy()
    q = np.stack([c & 15, c >> 4], axis=-1).reshape(len(c), -1)[:, :K].astype(np.int64) - 8
    return u.values(q, sc.float().cpu().numpy().astype(np.float64), group)


def _decode(cuda, steps, M, graph):
    """A tied 4-bit embedding / head with one 4-bit layer between, greedy, penalties on; returns the tokens and,
    step by step, the logits (before and after the rules) and the histories."""
    import torch

    import vvllm_b200 as v

    V, K, group = 1003, 256, 64
    emb = _quantized(cuda, make_weight(V, K, 1, 0.5), group)
    mlp = _quantized(cuda, make_weight(K, K, 2, 0.06), group)
    f16, i32 = torch.float16, torch.int32
    tok = torch.arange(M, device=cuda, dtype=i32) * 7 + 3
    x, h = torch.empty((M, K), dtype=f16, device=cuda), torch.empty((M, K), dtype=f16, device=cuda)
    raw, out = torch.empty((M, V), device=cuda), torch.empty((M, V), device=cuda)
    hist, hlen = torch.zeros((M, steps + 1), dtype=i32, device=cuda), torch.ones(M, dtype=i32, device=cuda)
    plen = torch.ones(M, dtype=i32, device=cuda)
    pen = [torch.full((M,), p, device=cuda) for p in (1.3, 0.2, 0.4)]
    mask = torch.full(((V + 31) // 32,), -1, dtype=i32, device=cuda)
    mask[3] = 0
    stream = torch.cuda.Stream()

    def step(s):
        v.dequantize_q4(x, *emb, group, rows=tok, stream=s)
        v.linear_q4_add(h, x, *mlp, group, None, x, stream=s)
        v.linear_q4(raw, h, *emb, group, stream=s)
        v.process_logits(out, raw, tok, history=hist, history_len=hlen, prompt_len=plen, repetition=pen[0],
                         presence=pen[1], frequency=pen[2], allowed=mask, stream=s)

    with torch.cuda.stream(stream):
        hist[:, 0] = tok
        start = tok.clone()
        step(stream)
        tok.copy_(start)
        g = torch.cuda.CUDAGraph()
        if graph:
            with torch.cuda.graph(g, stream=stream):
                step(stream)
        seen = []
        for i in range(steps):
            before = tok.clone()
            g.replay() if graph else step(stream)
            seen.append([t.clone() for t in (before, raw, out, tok, hist, hlen)])
            hist[:, i + 1] = tok
            hlen += 1
    torch.cuda.synchronize()
    return emb, mlp, group, K, V, [[t.cpu().numpy() for t in s] for s in seen], mask.cpu().numpy(), plen.cpu().numpy()


@pytest.mark.parametrize("M", [1, 3, 20])
def test_decode_steps_match_the_formulas(cuda, M):
    emb, mlp, group, K, V, seen, mask, plen = _decode(cuda, 6, M, graph=False)
    we, wm = _host_values(*emb, K, group), _host_values(*mlp, K, group)
    for before, raw, out, tok, hist, hlen in seen:
        x = we[before].astype(np.float16).astype(np.float64)
        h = (x @ wm.T + x).astype(np.float16).astype(np.float64)
        # h is rounded to fp16 from sums that may differ in their last bit: 2^-11 of it, times the head
        assert rowwise_normwise_err(raw, h @ we.T) <= 2e-3
        want, wtok = u.logits(raw, np.float32, history=hist, history_len=hlen, prompt_len=plen,
                              repetition=np.full(M, 1.3, np.float32), presence=np.full(M, 0.2, np.float32),
                              frequency=np.full(M, 0.4, np.float32), allowed=mask)
        assert np.array_equal(out, want) and np.array_equal(tok, wtok)
        assert not ((tok >= 96) & (tok < 128)).any()


@pytest.mark.parametrize("M", [1, 3, 20])
def test_decode_steps_replayed_from_a_graph(cuda, M):
    eager, graph = _decode(cuda, 6, M, graph=False)[5], _decode(cuda, 6, M, graph=True)[5]
    for a, b in zip(eager, graph):
        for x, y in zip(a, b):
            assert np.array_equal(x, y)


def _linear_inputs(cuda, M, N, K, seed):
    import torch

    r = np.random.default_rng(seed)
    q, s = r.integers(-8, 8, (N, K)), 2.0 ** r.integers(-2, 1, (N, K // 64))
    x = r.integers(-3, 4, (M, K)).astype(np.float64)
    return (torch.from_numpy(x).to(cuda).half(), torch.from_numpy(u.pack(q)).to(cuda),
            torch.from_numpy(u.bf16_bits(s).view(np.int16)).to(cuda).view(torch.bfloat16),
            u.linear(x, q, s, 64).astype(np.float32))


@pytest.mark.parametrize("M", [1, 8, 40])
def test_two_streams_at_once(cuda, M):
    """Calls on two streams, and replays of graphs captured on each, do not disturb one another."""
    import torch

    import vvllm_b200 as v

    streams, graphs, jobs = [torch.cuda.Stream(), torch.cuda.Stream()], [], []
    for i, st in enumerate(streams):
        x, q4, sc, want = _linear_inputs(cuda, M, 3000, 1024, 50 + i)
        out = torch.empty((M, 3000), device=cuda)
        tok = torch.empty(M, dtype=torch.int32, device=cuda)
        jobs.append((x, q4, sc, want, out, tok))
    torch.cuda.synchronize()

    def run(i):
        x, q4, sc, _, out, tok = jobs[i]
        v.linear_q4(out, x, q4, sc, 64, stream=streams[i])
        v.process_logits(None, out, tok, stream=streams[i])

    def check():
        torch.cuda.synchronize()
        for _, _, _, want, out, tok in jobs:
            assert np.array_equal(out.cpu().numpy(), want)
            assert np.array_equal(tok.cpu().numpy(), want.argmax(axis=1))
            out.fill_(float("nan"))
        torch.cuda.synchronize()

    for _ in range(20):
        run(0)
        run(1)
    check()
    for i, st in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            run(i)
        graphs.append(g)
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    check()


def test_a_graph_outlives_a_larger_call_on_its_stream(cuda):
    """The GEMM's scratch grows with a larger call; a graph captured before it still replays."""
    import torch

    import vvllm_b200 as v

    st = torch.cuda.Stream()
    x, q4, sc, want = _linear_inputs(cuda, 40, 500, 256, 9)
    out = torch.empty((40, 500), device=cuda)
    torch.cuda.synchronize()
    v.linear_q4(out, x, q4, sc, 64, stream=st)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        v.linear_q4(out, x, q4, sc, 64, stream=st)
    big = _linear_inputs(cuda, 24, 40000, 2048, 10)
    o2 = torch.empty((24, 40000), device=cuda)
    torch.cuda.synchronize()
    v.linear_q4(o2, *big[:3], 64, stream=st)
    out.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(o2.cpu().numpy(), big[3])


def test_graphs_of_one_stream_run_beside_each_other_and_beside_its_calls(cuda):
    """Graphs captured on one stream (the first calls there, so what they need is allocated during the captures)
    keep scratch of their own: replayed on other streams at once, beside calls on the stream of the capture."""
    import torch

    import vvllm_b200 as v

    st, others = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(3)]
    for again in range(3):  # graphs before are gone: their scratch is taken again
        jobs = [(*_linear_inputs(cuda, M, 2000, K, 60 + i), torch.empty((M, 2000), device=cuda))
                for i, (M, K) in enumerate([(40, 1024), (300, 2048), (40, 1024), (33, 4096)])]
        small = torch.empty((2, 2000), device=cuda)
        torch.cuda.synchronize()
        graphs = []
        for x, q4, sc, _, out in jobs[:3]:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                v.linear_q4(out, x, q4, sc, 64, stream=st)
                v.linear_q4(small, x[:2], q4, sc, 64, stream=st)
                v.linear_q4(out, x, q4, sc, 64, stream=st)
            graphs.append(g)
        for _ in range(30):
            for g, o in zip(graphs, others):
                with torch.cuda.stream(o):
                    g.replay()
            x, q4, sc, _, out = jobs[3]
            v.linear_q4(out, x, q4, sc, 64, stream=st)
        torch.cuda.synchronize()
        for x, q4, sc, want, out in jobs:
            assert np.array_equal(out.cpu().numpy(), want)
            out.fill_(float("nan"))
        del graphs, g


def test_copied_rows_in_graphs(cuda):
    """Calls whose rows are copied first: from graphs of one stream side by side, beside calls there."""
    import torch

    import vvllm_b200 as v

    st, others, jobs, graphs = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)], [], []
    for i, M in enumerate((1, 40, 6)):
        r = np.random.default_rng(i)
        q, s = r.integers(-8, 8, (500, 1021)), 2.0 ** r.integers(-2, 1, (500, 16))
        x = r.integers(-3, 4, (M, 1021)).astype(np.float64)
        jobs.append((torch.from_numpy(x).to(cuda).half(), torch.from_numpy(u.pack(q)).to(cuda),
                     torch.from_numpy(u.bf16_bits(s).view(np.int16)).to(cuda).view(torch.bfloat16),
                     u.linear(x, q, s, 64).astype(np.float32), torch.empty((M, 500), device=cuda)))
    torch.cuda.synchronize()
    for x, q4, sc, _, out in jobs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            v.linear_q4(out, x, q4, sc, 64, stream=st)
        graphs.append(g)
    for _ in range(20):
        for g, o in zip(graphs, others):
            with torch.cuda.stream(o):
                g.replay()
        v.linear_q4(jobs[2][4], *jobs[2][:3], 64, stream=st)
    torch.cuda.synchronize()
    for _, _, _, want, out in jobs:
        assert np.array_equal(out.cpu().numpy(), want)


def test_two_branches_of_one_capture(cuda):
    """Calls on two streams of one capture run beside each other in the graph."""
    import torch

    import vvllm_b200 as v

    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    jobs = [(*_linear_inputs(cuda, 40, 2000, 2048, 80 + i), torch.empty((40, 2000), device=cuda)) for i in range(2)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=a):
        b.wait_stream(a)
        for (x, q4, sc, _, out), s in zip(jobs, (a, b)):
            v.linear_q4(out, x, q4, sc, 64, stream=s)
        a.wait_stream(b)
    for _ in range(20):
        g.replay()
    torch.cuda.synchronize()
    for x, q4, sc, want, out in jobs:
        assert np.array_equal(out.cpu().numpy(), want)


def test_weights_used_right_after_they_are_written(cuda):
    """quantize, then linear, with nothing between: the linear call starts early and must not read ahead."""
    import torch

    import vvllm_b200 as v

    K, N = 1024, 4096
    x = torch.ones((1, K), dtype=torch.float16, device=cuda)
    xs = torch.ones((40, K), dtype=torch.float16, device=cuda)
    q4 = torch.empty((N, K // 2), dtype=torch.uint8, device=cuda)
    sc = torch.empty((N, K // 128), dtype=torch.bfloat16, device=cuda)
    ws = [torch.full((N, K), float(2.0 ** -i), device=cuda) for i in range(8)]
    outs = [torch.empty((1, N), device=cuda) for _ in ws]
    big = [torch.empty((40, N), device=cuda) for _ in ws]
    for w, o, b in zip(ws, outs, big):
        v.quantize_q4(w, q4, sc, 128)
        v.linear_q4(o, x, q4, sc, 128)
        v.linear_q4(b, xs, q4, sc, 128)
    torch.cuda.synchronize()
    for i, (o, b) in enumerate(zip(outs, big)):
        s = float(u.round_to_bf16(np.array([2.0 ** -i / 7]))[0])
        assert (o == 7 * s * K).all() and (b == 7 * s * K).all(), i


def test_rows_of_a_padded_batch(cuda):
    """Only the rows given are written: M of a larger buffer, and the tokens of finished rows stay."""
    import torch

    import vvllm_b200 as v

    for M in (1, 7, 30):
        x, q4, sc, want = _linear_inputs(cuda, M, 257, 512, 3 + M)
        buf = torch.full((M + 5, 257), -5.0, device=cuda)
        v.linear_q4(buf[:M], x, q4, sc, 64)
        tok = torch.full((M + 5,), 99, dtype=torch.int32, device=cuda)
        v.process_logits(buf[:M], buf[:M], tok[:M])
        torch.cuda.synchronize()
        assert np.array_equal(buf[:M].cpu().numpy(), want) and (buf[M:] == -5).all()
        assert np.array_equal(tok[:M].cpu().numpy(), want.argmax(axis=1)) and (tok[M:] == 99).all()


def test_empty_calls(cuda):
    import torch

    import vvllm_b200 as v

    q4 = torch.zeros((4, 32), dtype=torch.uint8, device=cuda)
    sc = torch.zeros((4, 1), dtype=torch.bfloat16, device=cuda)
    v.linear_q4(torch.empty((0, 4), device=cuda), torch.empty((0, 64), device=cuda), q4, sc, 64)
    v.linear_q4(torch.empty((2, 0), device=cuda), torch.empty((2, 64), device=cuda), q4[:0], sc[:0], 64)
    v.dequantize_q4(torch.empty((0, 64), device=cuda), q4, sc, 64, rows=torch.empty(0, dtype=torch.int32, device=cuda))
    v.quantize_q4(torch.empty((0, 64), device=cuda), q4[:0], sc[:0], 64)
    lg = torch.zeros((0, 50), device=cuda)
    v.process_logits(lg, lg, torch.empty(0, dtype=torch.int32, device=cuda))
    # lists without entries
    lg = torch.randn((2, 50), device=cuda)
    want = lg.clone()
    none = torch.empty((2, 0), dtype=torch.int32, device=cuda)
    v.process_logits(lg, lg, None, history=none, history_len=torch.zeros(2, dtype=torch.int32, device=cuda), bias_ids=none,
                     bias_values=torch.empty((2, 0), device=cuda), repetition=torch.full((2,), 2.0, device=cuda))
    assert torch.equal(lg, want)
    torch.cuda.synchronize()


def test_tensors_of_the_host_are_refused_beside_those_of_the_device(cuda):
    import torch

    import vvllm_b200 as v

    q4 = torch.zeros((4, 32), dtype=torch.uint8, device=cuda)
    sc = torch.zeros((4, 1), dtype=torch.bfloat16, device=cuda)
    x, out = torch.zeros((2, 64), device=cuda), torch.zeros((2, 4), device=cuda)
    for bad in ({"x": x.cpu()}, {"q4": q4.cpu()}, {"scales": sc.cpu()}, {"out": out.cpu()}, {"bias": torch.zeros(4)}):
        a = {"out": out, "x": x, "q4": q4, "scales": sc, "group": 64, **bad}
        with pytest.raises(ValueError, match="cpu"):
            v.linear_q4(**a)
    with pytest.raises(ValueError, match="cpu"):
        v.linear_q4_add(out, x, q4, sc, 64, None, out.cpu())
    with pytest.raises(ValueError, match="cpu"):
        v.process_logits(out, out, history=torch.zeros((2, 3), dtype=torch.int32),
                         history_len=torch.zeros(2, dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError, match="cpu"):
        v.dequantize_q4(x, q4, sc, 64, rows=torch.zeros(2, dtype=torch.int32))
