"""Embedding lookup and its gradient by sorted tokens, against the definition in 64 bits.

Tolerances follow from the arithmetic: a product or a sum in fp32 is off by at most ``u = 2**-24`` of its value
(fp64: ``2**-53``), a store in storage type ``t`` by ``finfo(t).eps / 2``, a sum of n terms by ``n * u`` of the sum
of their magnitudes, whatever its order.
"""
import pytest
import torch

from snn_gpu_training_bptt_amd import lif_cabi  # noqa: F401  (fails loudly without the built library)

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.float64, torch.bfloat16]


@pytest.fixture(scope="module")
def sf():
    from snn_gpu_training_bptt_amd import snnlib_func
    return snnlib_func


def unit(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def make(shape, V, C, dtype, seed, pad=0.0):
    gen = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, V, shape, generator=gen)
    if pad:
        tokens = torch.where(torch.rand(shape, generator=gen) < pad, -1, tokens)
    weight = torch.randn(V, C, generator=gen, dtype=torch.float64).to(dtype)
    grad = torch.randn(*shape, C, generator=gen, dtype=torch.float64).to(dtype)
    return tokens, weight, grad


def reference(tokens, weight, grad, scale):
    """(out, grad_weight, sum of |terms| of grad_weight, positions per row), all in 64 bits on the host."""
    V, C = weight.shape
    t, w, g = tokens.reshape(-1).long(), weight.double(), grad.double().reshape(-1, C)
    there = (t >= 0) & (t < V)
    out = torch.zeros(t.numel(), C, dtype=torch.float64)
    out[there] = scale * w[t[there]]
    gw, mag = (torch.zeros(V, C, dtype=torch.float64) for _ in range(2))
    gw.index_add_(0, t[there], scale * g[there])
    mag.index_add_(0, t[there], abs(scale) * g[there].abs())
    return out.reshape(*tokens.shape, C), gw, mag, torch.bincount(t[there], minlength=V).double()


def check(sf, tokens, weight, grad, scale=1.0):
    dtype, u = weight.dtype, unit(weight.dtype)
    half = torch.finfo(dtype).eps / 2
    w = weight.cuda().requires_grad_(True)
    y = sf.embed_func(tokens.cuda(), w, scale)
    (gw,) = torch.autograd.grad(y, w, grad.cuda())
    out_ref, gw_ref, mag, count = reference(tokens, weight, grad, scale)
    assert y.shape == out_ref.shape and y.dtype == dtype and gw.shape == weight.shape and gw.dtype == dtype
    # the scale rounded to the arithmetic type, the product, the store
    err = (y.detach().cpu().double() - out_ref).abs()
    assert bool((err <= out_ref.abs() * (2 * u + half) * 1.01).all()), float(err.max())
    # count sums, the scale, the product; the store
    bound = mag * ((count[:, None] + 3) * u) * 1.01 + gw_ref.abs() * half * 1.01
    err = (gw.cpu().double() - gw_ref).abs()
    assert bool((err <= bound).all()), float((err - bound).max())
    assert bool((gw.cpu()[count == 0] == 0).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape,V,C", [
    ((1, 1), 1, 1),                # one token, one row, one column
    ((1, 64), 32000, 1024),        # one generated token per sequence
    ((7, 3), 5, 3),                # rows of an odd number of bytes
    ((33, 5), 257, 250),           # two sorting workgroups, 8-byte accesses in fp32
    ((65, 1), 255, 8),             # one position more than a piece; V + 1 = 256 start entries
    ((64, 16), 256, 130),          # the last start entry belongs to a workgroup without rows
    ((300, 9), 11, 34),            # every row long
    ((40, 50), 3000, 2056),        # more columns than a workgroup holds
])
def test_lookup_and_gradient(sf, dtype, shape, V, C):
    check(sf, *make(shape, V, C, dtype, seed=V + C, pad=0.2), scale=0.37)


@gpu
@pytest.mark.parametrize("V,id_", [(1, 0), (700, 699), (200000, 131072)])
@pytest.mark.parametrize("n", [63, 64, 65, 128, 5000])
def test_every_position_holds_the_same_token(sf, V, id_, n):
    """The gradient of one row over pieces of 64 positions, up to tables sorted 1024 rows to a workgroup."""
    tokens, weight, grad = make((n, 1), V, 36, torch.float32, seed=n)
    check(sf, torch.full_like(tokens, id_), weight, grad, scale=1.5)


@gpu
def test_long_rows_begin_and_end_anywhere(sf):
    """Rows of 1 to 400 positions next to each other, in shuffled order: long rows that open a piece, close one,
    fill several, and share one."""
    gen = torch.Generator().manual_seed(3)
    counts = [1, 64, 65, 62, 66, 200, 3, 400, 64, 128, 129, 1, 70, 70, 70]
    tokens = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    tokens = tokens[torch.randperm(tokens.numel(), generator=gen)].reshape(-1, 1)
    grad = torch.randn(*tokens.shape, 50, generator=gen)
    check(sf, tokens, torch.randn(len(counts) + 2, 50, generator=gen), grad, scale=-2.0)


@gpu
def test_tokens_outside_the_table_are_no_tokens(sf):
    V = 10
    tokens = torch.tensor([[0, -1, V, 9], [-(2 ** 62), 2 ** 62, 2 ** 32 + 1, 5]])
    gen = torch.Generator().manual_seed(1)
    check(sf, tokens, torch.randn(V, 6, generator=gen), torch.randn(2, 4, 6, generator=gen))
    y = sf.embed_func(torch.full((3, 2), -1).cuda(), torch.full((V, 6), float("nan")).cuda())
    assert bool((y == 0).all())


@gpu
@pytest.mark.parametrize("shape", [(0, 4), (4, 0)])
def test_no_positions(sf, shape):
    w = torch.randn(5, 3, device="cuda", requires_grad=True)
    y = sf.embed_func(torch.zeros(shape, dtype=torch.long, device="cuda"), w)
    assert y.shape == shape + (3,)
    y.sum().backward()
    assert bool((w.grad == 0).all())


@gpu
def test_int32_tokens_strided_operands_and_shifted_storage(sf):
    tokens, weight, grad = make((12, 10), 40, 24, torch.float32, seed=5)
    t = tokens.int().t().contiguous().t().cuda()                    # int32, transposed in memory
    wide = torch.zeros(40, 31, device="cuda")
    wide[:, 3:27] = weight.cuda()                                  # rows 31 values apart, 12 bytes in
    g = torch.zeros(12 * 10 * 24 + 1, device="cuda")[1:].reshape(12, 10, 24).copy_(grad)   # 4 bytes off a boundary
    view = wide[:, 3:27].requires_grad_(True)
    y = sf.embed_func(t, view, 0.5)
    (gw,) = torch.autograd.grad(y, view, g)
    base = weight.cuda().requires_grad_(True)
    y0 = sf.embed_func(tokens.cuda(), base, 0.5)
    (gw0,) = torch.autograd.grad(y0, base, grad.cuda())
    assert torch.equal(y, y0) and torch.equal(gw, gw0)
    spread = weight.cuda().t().contiguous().t()                    # columns are the outer axis
    assert torch.equal(sf.embed_func(t, spread, 0.5), y0)


@gpu
def test_the_gradient_is_reproducible_and_independent_of_the_stream(sf):
    tokens, weight, grad = make((500, 20), 300, 64, torch.bfloat16, seed=8)
    t, g = (tokens % 7 * 41).cuda(), grad.cuda()
    first = sf.snnlib.embed_bp(t, g, 300, 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = sf.snnlib.embed_bp(t, g, 300, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)


@gpu
def test_gradient_against_differences(sf):
    tokens = torch.tensor([[3, 1], [3, -1], [0, 3]]).cuda()
    weight = torch.randn(5, 3, dtype=torch.float64, device="cuda", requires_grad=True)
    assert torch.autograd.gradcheck(lambda w: sf.embed_func(tokens, w, 0.7), (weight,))


@gpu
def test_captured_and_replayed(sf):
    tokens, weight, grad = make((90, 8), 50, 96, torch.float32, seed=11)
    t, w, g = tokens.cuda(), weight.cuda(), grad.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sf.snnlib.embed_bp(t, g, 50, 2.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = sf.snnlib.embed_fp(t, w, 2.0)
        gw = sf.snnlib.embed_bp(t, g, 50, 2.0)
    gen = torch.Generator().manual_seed(4)
    for _ in range(4):
        t.copy_(torch.randint(-1, 50, tokens.shape, generator=gen))
        graph.replay()
        want_y, want_gw = sf.snnlib.embed_fp(t, w, 2.0), sf.snnlib.embed_bp(t, g, 50, 2.0)
        torch.cuda.synchronize()
        assert torch.equal(y, want_y) and torch.equal(gw, want_gw)


@gpu
def test_second_derivatives_are_refused(sf):
    w = torch.randn(4, 3, device="cuda", requires_grad=True)
    y = sf.embed_func(torch.zeros(2, 2, dtype=torch.long, device="cuda"), w)
    (gw,) = torch.autograd.grad((y * y).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gw.sum(), w)


@gpu
def test_refusals(sf):
    w = torch.randn(4, 3, device="cuda")
    t = torch.zeros(2, 2, dtype=torch.long, device="cuda")
    for bad, match in [(lambda: sf.embed_func(t.float(), w), "int64 or int32"),
                       (lambda: sf.embed_func(t.cpu(), w), "ROCm GPU"),
                       (lambda: sf.embed_func(t, w.cpu()), "ROCm GPU"),
                       (lambda: sf.embed_func(t, w.half()), "unsupported dtype"),
                       (lambda: sf.embed_func(t, w[0]), "vocab, cout"),
                       (lambda: sf.embed_func(t, w[:0]), "at least one row"),
                       (lambda: sf.snnlib.embed_bp(t, w, 4, 1.0), "grad_out must be"),
                       (lambda: sf.snnlib.embed_bp(t, torch.zeros(2, 2, 3, device="cuda"), 0, 1.0), "vocab")]:
        with pytest.raises(RuntimeError, match=match):
            bad()


def test_a_host_tensor_is_refused(sf):
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        sf.embed_func(torch.zeros(2, 2, dtype=torch.long), torch.zeros(4, 3))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("C", [2, 5, 7, 9, 15, 17, 31, 33, 513, 2049])
def test_rows_that_start_and_end_inside_a_vector(sf, C, dtype):
    check(sf, *make((19, 5), 23, C, dtype, seed=C, pad=0.1), scale=-0.7)


@gpu
@pytest.mark.parametrize("shift", [1, 3])
def test_neighbours_of_rows_at_odd_addresses_stay_as_they_are(sf, shift):
    """The gradient written into storage one and three elements off a boundary, with values before and behind it."""
    from snn_gpu_training_bptt_amd import seq_cabi
    V, C, N = 11, 21, 37
    tokens, _, grad = make((N, 1), V, C, torch.bfloat16, seed=shift)
    held = torch.full((V * C + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = held[shift:shift + V * C].view(V, C)
    g = torch.zeros(N * C + shift, dtype=torch.bfloat16, device="cuda")[shift:].view(N, C)
    g.copy_(grad.reshape(N, C))
    need = seq_cabi.load().snnseq_embed_bp_workspace_bytes(2, N, V, C)
    seq_cabi.embed_bp_into(tokens.reshape(-1).cuda(), g, out, 1.0, torch.empty(need, dtype=torch.uint8, device="cuda"))
    plain = torch.zeros(V, C, dtype=torch.float64).index_add_(0, tokens.reshape(-1), grad.reshape(N, C).double())
    mag = torch.zeros(V, C, dtype=torch.float64).index_add_(0, tokens.reshape(-1), grad.reshape(N, C).double().abs())
    assert bool(((out.cpu().double() - plain).abs() <= mag * N * 2.0 ** -24 + plain.abs() * 2.0 ** -8).all())
    assert bool((held[:shift] == 7).all()) and bool((held[shift + V * C:] == 7).all())


@gpu
@pytest.mark.parametrize("n", [15, 16, 17, 31, 33, 8192, 8193])
def test_one_row_around_the_ends_of_pieces(sf, n):
    tokens, weight, grad = make((n, 1), 5, 12, torch.float32, seed=n)
    check(sf, torch.full_like(tokens, 3), weight, grad)


@gpu
def test_short_batches_of_long_rows_that_begin_and_end_anywhere(sf):
    gen = torch.Generator().manual_seed(8)
    counts = [1, 16, 17, 14, 18, 50, 3, 100, 16, 32, 33, 1, 20, 20, 20]
    tokens = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    tokens = tokens[torch.randperm(tokens.numel(), generator=gen)].reshape(-1, 1)
    grad = torch.randn(*tokens.shape, 50, generator=gen)
    check(sf, tokens, torch.randn(len(counts) + 2, 50, generator=gen), grad, scale=0.5)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V,C", [(50003, 40), (20001, 7), (17000, 1030)])
def test_large_tables_with_rows_of_every_length(sf, V, C, dtype):
    """Tables large enough that a group of threads sums several rows, with 0 to 200 tokens each and pad among them."""
    gen = torch.Generator().manual_seed(V)
    rows = torch.randperm(V, generator=gen)[:120]
    tokens = torch.repeat_interleave(rows, torch.randint(1, 40, (120,), generator=gen))
    tokens = torch.cat([tokens, torch.full((200,), int(rows[0])), torch.full((3,), V - 1), torch.zeros(2, dtype=torch.long),
                        torch.full((9,), -1)])
    tokens = tokens[torch.randperm(tokens.numel(), generator=gen)].reshape(-1, 1)
    grad = torch.randn(*tokens.shape, C, generator=gen).to(dtype)
    check(sf, tokens, torch.randn(V, C, generator=gen).to(dtype), grad, scale=0.5)


@gpu
def test_rows_whose_offset_passes_32_bits(sf):
    V, C = 4194500, 1024                                        # 4.3e9 values
    weight = torch.zeros(V, C, dtype=torch.bfloat16, device="cuda")
    weight[-2:] = torch.randn(2, C, device="cuda").bfloat16()
    weight.requires_grad_(True)
    tokens = torch.tensor([[V - 1], [V - 2], [0], [V - 1]], device="cuda")
    y = sf.embed_func(tokens, weight)
    assert torch.equal(y.detach(), weight.detach()[tokens])
    grad = torch.randn(4, 1, C, device="cuda").bfloat16()
    gw, = torch.autograd.grad(y, weight, grad)
    assert torch.equal(gw[-1], (grad[0, 0].float() + grad[3, 0].float()).bfloat16())
    assert torch.equal(gw[-2], grad[1, 0]) and torch.equal(gw[0], grad[2, 0])
    assert not bool(gw[1:-2].any())


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("V,C", [(9, 12), (50003, 40)])
@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan")])
def test_a_scale_that_is_not_finite_leaves_rows_without_a_token_zero(sf, scale, V, C, dtype):
    tokens = torch.tensor([[3, -1], [V - 1, V]]).cuda()
    w = torch.ones(V, C, dtype=dtype, device="cuda", requires_grad=True)
    y = sf.embed_func(tokens, w, scale)
    assert bool((y[0, 1] == 0).all()) and bool((y[1, 1] == 0).all())
    gw, = torch.autograd.grad(y, w, torch.ones_like(y))
    held = torch.zeros(V, dtype=torch.bool, device="cuda")
    held[[3, V - 1]] = True
    assert bool((gw[~held] == 0).all()) and not bool(gw[held].isfinite().any())
