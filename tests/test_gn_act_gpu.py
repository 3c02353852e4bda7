"""Group norm with an activation (channels last) against the definition in 64 bits.

Bounds are first-order error bounds of the formula, evaluated per value: with ``u = 2**-24`` (fp64: ``2**-53``) the
unit of the arithmetic and ``h = finfo(storage).eps / 2`` that of a store,
  * a sum of terms added along chains of at most CHAIN links is off by ``CHAIN * u`` of the sum of magnitudes.  A
    thread adds at most 32 values (16 positions times a vector of 8), a workgroup folds its rows in three steps
    of eight, and the columns of a group follow: below 128 for every size here.  Parameter sums go on over the
    samples and over 32 + 32 partial rows: below 256;
  * the variance is ``CHAIN * u`` plus four roundings, its inverse root half of that plus three;
  * an activation's slope is at most 1.13 and changes by at most 1.2 per unit of z; evaluating it costs 16 ``u`` of
    ``1 + |z|`` (exponential, error function and reciprocal are good to a few units in the last place).  The slope
    of the relu jumps where |z| is below the bound of z.
"""
import math

import pytest
import torch

from snn_gpu_training_bptt_amd import lif_cabi  # noqa: F401

gpu = pytest.mark.gpu
EPS = 1e-5
CHAIN, CHAIN_PARAMS = 128, 256
ACTS = ["none", "relu", "silu", "gelu"]
DTYPES = [torch.float32, torch.float64, torch.bfloat16]


@pytest.fixture(scope="module")
def sf():
    from snn_gpu_training_bptt_amd import snnlib_func
    return snnlib_func


def act_and_slope(z, act):
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def with_bounds(x, w, b, gy, groups, act):
    """((y, grad_x, grad_w, grad_b), their bounds) in 64 bits."""
    u = 2.0 ** -53 if x.dtype == torch.float64 else 2.0 ** -24
    half = torch.finfo(x.dtype).eps / 2
    shape, C = x.shape, x.shape[-1]
    X, GY = (t.double().reshape(shape[0] * shape[1], -1, groups, C // groups) for t in (x, gy))
    W, B = (t.double().reshape(1, 1, groups, -1) for t in (w, b))
    mean_of = lambda t: t.mean(dim=(1, 3), keepdim=True)
    m = mean_of(X)
    var = mean_of((X - m) ** 2)
    r = (var + EPS).rsqrt()
    xhat = (X - m) * r
    d_m = CHAIN * u * mean_of(X.abs())
    d_r = (CHAIN / 2 + 8) * u + (d_m * r) ** 2             # relative; a wrong mean enters the variance squared
    d_xhat = xhat.abs() * (d_r + 2 * u) + r * (d_m + u * (X - m).abs())
    z = xhat * W + B
    d_z = W.abs() * d_xhat + 2 * u * ((xhat * W).abs() + B.abs())
    y, slope = act_and_slope(z, act)
    d_act = 16 * u * (1 + z.abs()) if act in ("silu", "gelu") else 0.0
    b_y = 1.13 * d_z + d_act * (z.abs() + 1) + half * y.abs()
    d_slope = torch.where(z.abs() <= d_z, 1.0, 0.0) if act == "relu" else 1.2 * d_z * (act != "none") + d_act
    gz = GY * slope
    d_gz = GY.abs() * d_slope + u * gz.abs()
    c1, c2 = mean_of(gz * W), mean_of(gz * W * xhat)
    d_c1 = CHAIN * u * mean_of((gz * W).abs()) + mean_of(d_gz * W.abs())
    d_c2 = CHAIN * u * mean_of((gz * W * xhat).abs()) + mean_of((d_gz * xhat.abs() + gz.abs() * d_xhat) * W.abs())
    inner = (gz * W).abs() + c1.abs() + (xhat * c2).abs()
    gx = r * (gz * W - c1 - xhat * c2)
    b_gx = r * (d_gz * W.abs() + d_c1 + xhat.abs() * d_c2 + c2.abs() * d_xhat + (d_r + 4 * u) * inner) + half * gx.abs()
    total = lambda t: t.sum(dim=(0, 1)).reshape(C)
    gw, gb = total(gz * xhat), total(gz)
    b_gw = CHAIN_PARAMS * u * total((gz * xhat).abs()) + total(d_gz * xhat.abs() + gz.abs() * d_xhat) + half * gw.abs()
    b_gb = CHAIN_PARAMS * u * total(gz.abs()) + total(d_gz) + half * gb.abs()
    return (y.reshape(shape), gx.reshape(shape), gw, gb), (b_y.reshape(shape), b_gx.reshape(shape), b_gw, b_gb)


def make(shape, dtype, seed, offset=0.5):
    gen = torch.Generator().manual_seed(seed)
    C = shape[-1]
    rand = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    x = rand(*shape) * (0.5 + rand(C).abs()) + offset * rand(C)
    return tuple(t.to(dtype) for t in (x, 1 + 0.3 * rand(C), 0.2 * rand(C), rand(*shape)))


def run(sf, x, w, b, gy, groups, act):
    x, w, b = (t.cuda().requires_grad_(True) for t in (x, w, b))
    y = sf.gn_act_func(x, w, b, groups, EPS, act)
    return (y.detach(),) + torch.autograd.grad(y, (x, w, b), gy.cuda())


def check(sf, shape, groups, act, dtype, seed=0, offset=0.5):
    args = make(shape, dtype, seed, offset)
    got = run(sf, *args, groups, act)
    want, bounds = with_bounds(*args, groups, act)
    for a, e, bound, what in zip(got, want, bounds, ("y", "grad_x", "grad_weight", "grad_bias")):
        assert a.dtype == dtype and a.shape == e.shape
        err = (a.cpu().double() - e).abs()
        # products of two errors are left out of the bounds: 5 % on top, and nothing below the smallest number
        over = err - (1.05 * bound + 1e-37)
        assert bool((over <= 0).all()), f"{what}: off by {float(err.max())}, {float(over.max())} over its bound"


SHAPES = [  # (shape, groups): which layout they take
    ((1, 32, 512), 8),             # rows: one token per sequence
    ((3, 5, 24), 1),               # rows: one group
    ((2, 3, 7), 7),                # rows: groups of one value (variance 0)
    ((4, 3, 90), 9),               # rows: ten channels
    ((9, 7, 1536), 3),             # rows: two and four vectors per lane
    ((2, 70, 1022), 2),            # rows: 511 channels
    ((2, 2, 4100), 1),             # slab with a single position: a group too wide for the rows layout
    ((3, 2, 13, 11, 90), 9),       # slab: odd planes
    ((2, 2, 5, 64), 4),            # slab: one spatial axis
    ((2, 3, 32, 32, 128), 32),     # slab in workgroups of 1024
    ((1, 2, 3, 2, 6), 2),          # slab: tiny
    ((1, 5, 1, 2, 3, 9), 3),       # slab: three spatial axes
    ((1, 2, 70, 71, 48), 3),       # split
    ((2, 1, 64, 64, 33), 1),       # split: odd rows of 33 channels
    ((1, 1, 3000, 2100), 4),       # split: several column blocks
]


@gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_against_the_definition(sf, shape, groups, dtype, act):
    check(sf, shape, groups, act, dtype, seed=len(shape) + groups)


@gpu
@pytest.mark.parametrize("shape,groups", [((3, 700, 64), 4), ((40, 100, 2, 2, 32), 8), ((2050, 1, 40), 5)])
def test_parameter_gradients_over_many_samples(sf, shape, groups):
    check(sf, shape, groups, "silu", torch.float32, seed=1)


@gpu
@pytest.mark.parametrize("shape,groups", [((2, 3, 256), 4), ((2, 2, 9, 9, 32), 4), ((1, 1, 80, 80, 32), 2)])
def test_a_mean_far_from_zero(sf, shape, groups):
    """Values around 1e3 with a spread of one: the variance is taken around the mean, not from squares."""
    check(sf, shape, groups, "none", torch.float32, seed=2, offset=1e3 / 0.8)


@gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,groups", [((2, 3, 10), 2), ((1, 2, 3, 3, 4), 2)])
def test_gradients_against_differences(sf, shape, groups, act):
    x, w, b, _ = (t.cuda().requires_grad_(True) for t in make(shape, torch.float64, seed=3))
    assert torch.autograd.gradcheck(lambda *a: sf.gn_act_func(*a, groups, EPS, act), (x, w, b))


@gpu
@pytest.mark.parametrize("shape,groups", [((2, 3, 64), 4), ((2, 2, 6, 6, 16), 4), ((1, 1, 80, 80, 32), 2)])
def test_strided_operands_shifted_storage_and_expanded_gradients(sf, shape, groups):
    x, w, b, gy = make(shape, torch.float32, seed=4)
    want = run(sf, x, w, b, gy, groups, "silu")
    apart = torch.zeros(shape[:-1] + (shape[-1] + 3,), device="cuda")
    apart[..., 3:] = x.cuda()
    shifted = torch.zeros(x.numel() + 1, device="cuda")[1:].view(shape).copy_(x)      # 4 bytes off a boundary
    firsts = torch.stack([w, b]).t().contiguous().cuda()                              # weight and bias interleaved
    for view in (apart[..., 3:], shifted, x.cuda().transpose(0, 1).contiguous().transpose(0, 1)):
        got = run(sf, view, firsts[:, 0], firsts[:, 1], gy, groups, "silu")
        for a, e in zip(got, want):
            # another access width adds in another order: both lie within their bounds
            torch.testing.assert_close(a, e, rtol=1e-4, atol=1e-4)
    one = gy[:1].expand(shape)
    for a, e in zip(run(sf, x, w, b, one, groups, "silu"), run(sf, x, w, b, one.contiguous(), groups, "silu")):
        assert torch.equal(a, e)


@gpu
def test_channels_last_images_are_taken_as_they_lie(sf):
    """A ``[T*B, C, H, W]`` tensor in channels-last memory is a dense ``[T, B, H, W, C]`` view: same values as torch's
    own group norm over the channel axis."""
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(4, 32, 5, 7, generator=gen).cuda().contiguous(memory_format=torch.channels_last)
    w, b = torch.randn(32, generator=gen).cuda(), torch.randn(32, generator=gen).cuda()
    view = x.permute(0, 2, 3, 1).reshape(2, 2, 5, 7, 32)
    assert view.data_ptr() == x.data_ptr()
    y = sf.gn_act_func(view, w, b, 8, EPS, "relu").reshape(4, 5, 7, 32).permute(0, 3, 1, 2)
    torch.testing.assert_close(y, torch.relu(torch.nn.functional.group_norm(x, 8, w, b, EPS)), rtol=1e-5, atol=1e-5)


@gpu
@pytest.mark.parametrize("shape,groups", [((2, 3, 64), 4), ((2, 2, 6, 6, 16), 4), ((1, 1, 80, 80, 32), 2)])
def test_values_that_are_not_finite_stay_in_their_group(sf, shape, groups):
    x, w, b, gy = make(shape, torch.float32, seed=7)
    clean = run(sf, x, w, b, gy, groups, "silu")[0]
    x = x.clone()
    x[0, 0, ..., 0] = float("nan")
    x[0, 1 % shape[1], ..., -1] = float("inf")
    y = run(sf, x, w, b, gy, groups, "silu")[0]
    per = shape[-1] // groups
    touched = torch.zeros(shape, dtype=torch.bool)
    touched[0, 0, ..., :per] = True
    touched[0, 1 % shape[1], ..., -per:] = True
    assert bool(torch.isnan(y.cpu()[touched]).all())
    assert torch.equal(y.cpu()[~touched], clean.cpu()[~touched])


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activations_far_out(sf, act):
    """|z| up to 1e4: the slope is 0 or 1 there, never inf * 0."""
    x = torch.tensor([-1.0, 1.0, -1.0, 1.0]).reshape(1, 1, 4)
    w, b = torch.full((4,), 1e4), torch.zeros(4)
    y, gx, gw, gb = run(sf, x, w, b, torch.ones(1, 1, 4), 1, act)
    assert bool(torch.isfinite(torch.cat([t.flatten() for t in (y, gx, gw, gb)])).all())
    assert gb.cpu().tolist() == [0.0, 1.0, 0.0, 1.0] and float(y[0, 0, 0]) == 0.0


@gpu
@pytest.mark.parametrize("shape", [(0, 3, 8), (3, 0, 4, 4, 8)])
def test_an_empty_batch(sf, shape):
    y, gx, gw, gb = run(sf, *make(shape, torch.float32, 0), 2, "silu")
    assert y.shape == shape and gx.shape == shape and bool((gw == 0).all()) and bool((gb == 0).all())


@gpu
@pytest.mark.parametrize("shape,groups", [((64, 9, 128), 4), ((2, 9, 6, 6, 16), 4), ((1, 1, 80, 80, 32), 2)])
def test_captured_replayed_and_on_another_stream(sf, shape, groups):
    x, w, b, gy = (t.cuda() for t in make(shape, torch.float32, seed=9))

    def step():
        mean, rstd, y = sf.snnlib.gn_act_fp(x, w, b, groups, EPS, "gelu")
        return [y] + sf.snnlib.gn_act_bp(x, w, b, mean, rstd, groups, "gelu", gy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, e) for a, e in zip(other, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        x.mul_(1.01).add_(0.1 * k)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, want))


@gpu
def test_refusals(sf):
    x, w, b, _ = (t.cuda() for t in make((2, 2, 8), torch.float32, 0))
    f = lambda *a: sf.gn_act_func(*a)
    for bad, match in [(lambda: f(x, w, b, 3, EPS, "none"), "must divide the channels"),
                       (lambda: f(x, w, b, 0, EPS, "none"), "must divide the channels"),
                       (lambda: f(x, w, b, 2, EPS, "tanh"), "unknown activation"),
                       (lambda: f(x, w, b, 2, -1.0, "none"), "must not be negative"),
                       (lambda: f(x[0], w, b, 2, EPS, "none"), r"\[T, B, ..., C\]"),
                       (lambda: f(x, w[:4], b, 2, EPS, "none"), "one value per channel"),
                       (lambda: f(x, w, b.double(), 2, EPS, "none"), "dtype of x"),
                       (lambda: f(x, w, b.cpu(), 2, EPS, "none"), "ROCm GPU"),
                       (lambda: f(x.half(), w.half(), b.half(), 2, EPS, "none"), "unsupported dtype"),
                       (lambda: f(x.reshape(2, 2, 1, 8)[:, :, :0], w, b, 2, EPS, "none"), "no values per group")]:
        with pytest.raises(RuntimeError, match=match):
            bad()
    mean, rstd, _ = sf.snnlib.gn_act_fp(x, w, b, 2, EPS, "none")
    with pytest.raises(RuntimeError, match="what gn_act_fp returned"):
        sf.snnlib.gn_act_bp(x, w, b, mean[..., :1], rstd, 2, "none", x)
    with pytest.raises(RuntimeError, match="same shape"):
        sf.snnlib.gn_act_bp(x, w, b, mean, rstd, 2, "none", x[:1])


def test_a_host_tensor_is_refused(sf):
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        sf.gn_act_func(torch.zeros(2, 2, 4), torch.ones(4), torch.zeros(4), 2)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("channels", [1, 6, 24, 128])
def test_a_group_of_one_value_has_no_input_gradient(sf, channels, act, dtype):
    """The value is its own mean: y is act(bias), and grad_y * w minus its mean over one value is exactly 0."""
    gen = torch.Generator().manual_seed(channels)
    x, gy = (torch.randn(7, 3, channels, generator=gen).to(dtype).cuda() for _ in range(2))
    w, b = (torch.randn(channels, generator=gen).to(dtype).cuda() for _ in range(2))
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = sf.gn_act_func(x, w, b, channels, EPS, act)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
    assert torch.equal(y, y[:1, :1].expand_as(y))
    assert torch.equal(gx, torch.zeros_like(gx))
    assert torch.equal(gw, torch.zeros_like(gw))


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape,groups", [
    ((9, 3, 3 * 5), 3),              # rows: a vector and one value of the next
    ((9, 3, 2 * 111), 2),
    ((3, 2, 6, 5, 4 * 3), 4),        # slab: groups narrower than a vector
    ((5, 3, 11, 20, 9 * 43), 9),     # slab of 1024 threads
    ((1, 2, 60, 70, 2 * 13), 2),     # split
])
def test_groups_that_end_inside_a_vector(sf, shape, groups, dtype):
    check(sf, shape, groups, "silu", dtype, seed=groups)


@gpu
@pytest.mark.parametrize("shape,groups", [((3, 2, 2 * 7), 2), ((2, 2, 6, 6, 3 * 5), 3), ((1, 1, 80, 80, 2 * 11), 2)])
def test_values_that_are_not_finite_stay_in_their_group_where_vectors_overlap(sf, shape, groups):
    x, w, b, gy = (t.cuda() for t in make(shape, torch.float32, 3))
    first = run(sf, x, w, b, gy, groups, "silu")
    cpg = shape[-1] // groups
    bad = x.clone()
    bad.reshape(-1, shape[-1])[0, cpg - 1] = float("nan")      # the last value of the first sample's first group
    second = run(sf, bad, w, b, gy, groups, "silu")
    for a, c in zip(first[:2], second[:2]):
        a, c = (t.reshape(shape[0] * shape[1], -1, groups, cpg) for t in (a, c))
        assert bool(c[0, :, 0].isnan().all())
        assert torch.equal(a[0, :, 1:], c[0, :, 1:]) and torch.equal(a[1:], c[1:])


@gpu
@pytest.mark.parametrize("shape,groups", [((2, 33000, 65536), 64), ((3, 1400, 16, 16, 4096), 64), ((1, 270, 128, 128, 1024), 4)])
def test_samples_whose_offset_passes_32_bits(sf, shape, groups):
    """Rows, slab and split layouts over more than 2**32 values: the first and the last sample by themselves."""
    C = shape[-1]
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_()
    w, b = 1 + 0.1 * torch.randn(C, device="cuda").bfloat16(), 0.1 * torch.randn(C, device="cuda").bfloat16()
    x.requires_grad_(True)
    y = sf.gn_act_func(x, w, b, groups, EPS, "silu")
    gx, = torch.autograd.grad(y, x, x.detach())
    for t, s in ((0, 0), (shape[0] - 1, shape[1] - 1)):
        one = x.detach()[t:t + 1, s:s + 1]
        (y_ref, gx_ref, _, _), (b_y, b_gx, _, _) = with_bounds(one.cpu(), w.cpu(), b.cpu(), one.cpu(), groups, "silu")
        for a, e, bound in ((y.detach(), y_ref, b_y), (gx, gx_ref, b_gx)):
            err = (a[t:t + 1, s:s + 1].cpu().double() - e).abs()
            assert bool((err <= 1.05 * bound + 1e-37).all())
