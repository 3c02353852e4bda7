"""The token layers at sizes where their kernels go round their loops, against 64 bits: several samples per lane and per
workgroup in the group norm, pieces of 32 positions and rows that a wavefront cannot keep in the embedding's gradient,
a hundred chunks in the gated delta rule.  Bounds are those of the tests of each operator."""
import pytest
import torch

from snn_gpu_training_bptt_amd import lif_cabi  # noqa: F401
import test_embed_gpu
import test_gated_delta_gpu as delta
import test_gn_act_gpu as gn

pytestmark = pytest.mark.gpu
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16


@pytest.fixture(scope="module")
def sf():
    from snn_gpu_training_bptt_amd import snnlib_func
    return snnlib_func


@pytest.mark.parametrize("shape,groups,dtype,act", [
    # rows, one vector per lane: four samples requested together forward (the last group has fewer), eight of each lane backward
    ((16387, 1, 32 * 16), 32, F32, "silu"),
    ((16386, 1, 32 * 24), 32, BF16, "gelu"),
    ((5463, 3, 32 * 20), 32, BF16, "silu"),              # 16389 samples, groups that end inside a vector
    ((16385, 1, 32 * 6), 32, F64, "silu"),
    ((2049, 8, 32 * 5), 32, F64, "none"),                # 16392
    # rows, two and four vectors per lane
    ((3001, 1, 3 * 512), 3, F32, "silu"),
    ((9003, 1, 1021), 1, F32, "gelu"),
    # slab in workgroups of 1024, the next sample requested ahead: 300 samples on 64 of them
    ((10, 30, 32, 32, 128), 32, F32, "silu"),
    # slab in workgroups of 256: 5000 samples on 2048, groups that end inside a vector
    ((50, 100, 5, 5, 26), 2, F32, "relu"),
    ((50, 100, 5, 5, 26), 2, BF16, "silu"),
])
def test_group_norm_of_many_samples(sf, shape, groups, dtype, act):
    """Chains of a channel's sum: up to eight samples of a lane, the lanes that share the channel (up to 32), at most
    2048 / 32 partial rows and 32 of their sums: below the 256 links that the bounds count."""
    gen = torch.Generator(device="cuda").manual_seed(groups)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=torch.float64)
    C = shape[-1]
    args = [t.to(dtype) for t in (rand(*shape) * (0.5 + rand(C).abs()) + 0.5 * rand(C), 1 + 0.3 * rand(C), 0.2 * rand(C),
                                  rand(*shape))]
    got = gn.run(sf, *args, groups, act)
    want, bounds = gn.with_bounds(*args, groups, act)
    for a, e, bound, what in zip(got, want, bounds, ("y", "grad_x", "grad_weight", "grad_bias")):
        assert a.dtype == dtype and a.shape == e.shape
        over = (a.double() - e).abs() - (1.05 * bound + 1e-37)
        assert bool((over <= 0).all()), f"{what}: {float(over.max())} over its bound"


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("V", [3000, 140000])
@pytest.mark.parametrize("n", [9001, 33000])
def test_embedding_gradient_of_frequent_and_rare_tokens(sf, n, V, dtype):
    """Pieces of 32 positions: rows of 1 to 200 around their multiples, in any order, so that long rows begin, end, share
    and fill pieces.  Two fifths of the tokens fall on ten neighbouring rows: of those a wavefront of the sort meets more
    than it keeps, from several rows.  Tables of which a sorting workgroup has 256 rows, and 1024."""
    gen = torch.Generator().manual_seed(n + V)
    lengths = torch.tensor([31, 32, 33, 63, 64, 65, 96, 1, 2, 200, 30, 34] * 6)
    rows = torch.randperm(V - 512, generator=gen)[:len(lengths)] + 512
    tokens = torch.repeat_interleave(rows, lengths)
    hot = 300 + torch.randint(0, 10, (2 * n // 5,), generator=gen)
    rest = n - tokens.numel() - hot.numel()
    tokens = torch.cat([tokens, hot, torch.randint(-40, V + 40, (rest,), generator=gen)])
    tokens = tokens[torch.randperm(n, generator=gen)].reshape(-1, 1)
    grad = torch.randn(n, 1, 20, generator=gen).to(dtype)
    test_embed_gpu.check(sf, tokens, torch.randn(V, 20, generator=gen).to(dtype), grad, scale=0.75)


@delta.both
@pytest.mark.parametrize("lengths", [None, [8197, 5000]])
def test_gated_delta_gradients_over_a_hundred_chunks(sf, lengths, dtype):
    delta.check(sf, 8197, 2, 1, 2, 24, 16, dtype, seed=3, lengths=lengths)


@delta.both
def test_gated_delta_prompt_of_a_hundred_chunks(sf, dtype):
    T = 8192
    x, _, _ = delta.make(T, 1, 1, 2, 128, 128, dtype, seed=4)
    with torch.no_grad():
        o, last = sf.gated_delta_func(*(x[n].cuda() for n in delta.NAMES), None, 0.1)
    want_o, want_last = delta.recurrence({n: t.double() for n, t in x.items()}, None, 0.1)
    delta.compare({"o": o, "last": last}, {"o": want_o, "last": want_last}, T, dtype)
