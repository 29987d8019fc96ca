"""Activations far larger than their neighbours, as models have them in a few channels: where a weight row has the
value 0 at those, its output is the others' sum, and loses no more than the header of the C interface says."""
import pytest

pytestmark = pytest.mark.gpu


def _values(q4, sc, K, group):
    import torch

    q = torch.stack((q4 & 15, q4 >> 4), dim=-1).flatten(1)[:, :K].double() - 8
    return q * sc.double().repeat_interleave(group, dim=1)[:, :K]


@pytest.mark.parametrize("big", [1000.0, 30000.0])
@pytest.mark.parametrize("xdt,M", [("float16", 1), ("float16", 2), ("float16", 3), ("float16", 12), ("float32", 1),
                                   ("float32", 2), ("float32", 3), ("float32", 8), ("float32", 20)])
@pytest.mark.parametrize("N,K,group", [(300, 1024, 32), (70, 18944, 128), (500, 1000, 64), (1000, 160, 64)])
def test_neighbours_of_massive_activations(cuda, N, K, group, xdt, M, big):
    """Tolerance.  Three to sixteen fp16 tokens are used as they are; one or two, and fp32 ones, are rounded by at most
    2^-22 of the largest of their 128 neighbours, which is `big` in the first five such chunks (elsewhere 2^-22 of 0.06,
    below what the sums lose).  The sums: an output's terms, taken apart into signed digits, add up to at most 3 * size
    in magnitude (size = sum |x w|, of the inputs as rounded; a digit is at most half the next one's step, so 128 =
    256 - 128 is the worst).  Each of a warp's fp32 operations (a group's sum times its scale, the chunk's, the
    running sum: three a group, and 64 to join warps and ranks) is off by 2^-24 of that."""
    import torch

    import vvllm_b200 as v

    g = torch.Generator(device=cuda).manual_seed(K + M)
    q4 = torch.randint(0, 256, (N, (K + 1) // 2), dtype=torch.uint8, device=cuda, generator=g)
    sc = (0.01 + 0.01 * torch.rand((N, -(-K // group)), device=cuda, generator=g)).bfloat16()
    x = 0.01 * torch.randn((M, K), device=cuda, generator=g)
    at = torch.arange(6, K, 128, device=cuda)[:5]  # one a chunk, in the first five
    x[:, at] = big * torch.where(torch.rand((M, len(at)), device=cuda, generator=g) < 0.5, -1.0, 1.0)
    q4[:, at // 2] = (q4[:, at // 2] & 0xF0) | 8
    x = x.to(getattr(torch, xdt))
    w = _values(q4, sc, K, group)
    assert (w[:, at] == 0).all()
    y, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    out = torch.empty((M, N), device=cuda)
    v.linear_q4(out, x, q4, sc, group)
    cut = 0.0 if xdt == "float16" and M > 2 else 2.0 ** -22 * big * w.abs()[:, :640].sum(dim=1)
    bound = cut + (3 * (K // 32 + 1) + 64) * 3 * 2.0 ** -24 * (size + cut)
    err = (out.double() - y).abs()
    assert (err <= bound).all(), float((err / bound).max())
    assert v.kernel_error() == 0


@pytest.mark.parametrize("xdt", ["float16", "float32"])
def test_one_sequence_beside_a_batch(cuda, xdt):
    """The same token alone, in a pair, and among twelve: without large ones the errors are those of fp32 sums."""
    import torch

    import vvllm_b200 as v

    N, K, group = 2000, 3584, 128
    g = torch.Generator(device=cuda).manual_seed(3)
    q4 = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=cuda, generator=g)
    sc = (0.01 + 0.01 * torch.rand((N, K // group), device=cuda, generator=g)).bfloat16()
    x = torch.randn((12, K), device=cuda, generator=g).to(getattr(torch, xdt))
    y = x.double() @ _values(q4, sc, K, group).T
    for M in (1, 2, 12):
        out = torch.empty((M, N), device=cuda)
        v.linear_q4(out, x[:M], q4, sc, group)
        # sums of K / group = 28 group sums, rounded to 2^-24 of themselves: sqrt(28) * 2^-24 of the result's deviation,
        # twice that for their scales and the joins; an input is off by 2^-23 of 2^3 at most (no input is above 8),
        # over sqrt(3) on average, of its deviation 1
        assert x.abs().max() < 8
        cut = 0.0 if xdt == "float16" and M > 2 else 2.0 ** -20 / 3 ** 0.5
        assert float((out.double() - y[:M]).norm() / y[:M].norm()) <= 2 * 28 ** 0.5 * 2.0 ** -24 + cut
