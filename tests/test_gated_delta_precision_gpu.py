"""The gated delta rule holds what lies between its inputs and its results to 24 bits, whatever the storage type.

A value of 16 bits (two bf16 numbers) in its place would pass a test by norm.  Here every result is the difference of two
nearly equal terms that follow from the inputs in a few operations: x, and its first two bf16 parts.  What is left is the
part of x that 16 bits do not hold, up to 2**-17.  A case has 256 of them, one per head.

Tolerance, derived: every term is at most one, and on its way it is rounded at most 16 times in fp32 -- the exponential (a
unit in the last place and its argument's rounding, 4), the products with a rate, a decay and the scale (3), the additions
of the three parts of either term to a sum (6), the difference itself and the conversion from parts (3).  Each is off by at
most 2**-24, so a result by 16 * 2**-24 = 2**-20 and half a step of its storage type.  References are 64-bit.
"""
import pytest
import torch

from snn_gpu_training_bptt_amd import lif_cabi  # noqa: F401
from test_gated_delta_gpu import NAMES, recurrence

pytestmark = pytest.mark.gpu
B, H = 16, 16
BOUND = 2.0 ** -20


@pytest.fixture(scope="module")
def sf():
    from snn_gpu_training_bptt_amd import snnlib_func
    return snnlib_func


def coarse(x):
    """The first two bf16 parts of fp32 values."""
    first = x.bfloat16().float()
    return first + (x - first).bfloat16().float()


def values(seed):
    """fp32 values in (1/2, 1), one per head."""
    return 0.5 + 0.5 * torch.rand(B, H, generator=torch.Generator().manual_seed(seed))


def blank():
    """Operands of three steps that do nothing, gradients of zero."""
    zero, T, Dk, Dv = torch.zeros, 3, 4, 2
    x = {"q": zero(T, B, H, Dk), "k": zero(T, B, H, Dk), "v": zero(T, B, H, Dv), "g": zero(T, B, H),
         "beta": zero(T, B, H), "state": zero(B, H, Dk, Dv)}
    return x, zero(T, B, H, Dv), zero(B, H, Dk, Dv)


def orthogonal_keys(x):
    """Two keys of length sqrt(1/2) whose first components cancel."""
    x["k"][0, ..., 0] = x["k"][0, ..., 1] = x["k"][1, ..., 1] = 0.5
    x["k"][1, ..., 0] = -0.5


def state_in_output(x, go, gs):            # o = q . S
    a = values(0)
    x["state"][..., 0, 0], x["state"][..., 1, 0] = a, coarse(a)
    x["q"][0, ..., 0], x["q"][0, ..., 1] = 1, -1
    return "o", (0, ..., 0)


def rows_in_output(x, go, gs):             # o = P R with R = beta v
    a = values(1)
    x["beta"][0], x["beta"][1] = a, coarse(a)
    x["v"][..., 0] = 1
    x["k"][0, ..., 0] = x["k"][1, ..., 1] = 1
    x["q"][1, ..., 0], x["q"][1, ..., 1] = 1, -1
    return "o", (1, ..., 0)


def decay_in_output(x, go, gs):            # o = P R with P = e^g
    a = values(2)
    x["g"][1] = a.log()
    x["beta"][0], x["beta"][1] = 1, coarse(a)
    x["v"][..., 0] = 1
    x["k"][0, ..., 0] = x["k"][1, ..., 1] = 1
    x["q"][1, ..., 0], x["q"][1, ..., 1] = 1, -1
    return "o", (1, ..., 0)


def scores_in_grad_q(x, go, gs):           # dQ = N K with N = dO R^T
    a = values(3)
    x["beta"][0], x["beta"][1] = a, coarse(a)
    x["v"][..., 0] = 1
    orthogonal_keys(x)
    go[1, ..., 0] = 1
    return "grad_q", (1, ..., 0)


def state_in_grad_q(x, go, gs):            # dQ = S dO
    a = values(4)
    x["state"][..., 0, 0], x["state"][..., 0, 1] = a, coarse(a)
    go[0, ..., 0], go[0, ..., 1] = 1, -1
    return "grad_q", (0, ..., 0)


def scores_in_grad_k(x, go, gs):           # dK = N^T Q
    a = values(5)
    x["beta"][0] = a
    x["g"][1] = (coarse(a) / a).log()
    x["v"][0, ..., 0] = 1
    x["k"][0, ..., 0] = x["k"][1, ..., 1] = 1
    x["q"][0, ..., 2], x["q"][1, ..., 2] = 0.5, -0.5
    go[..., 0] = 1
    return "grad_k", (0, ..., 2)


def corrections_in_grad_k(x, go, gs):      # dK = M^T K with M = -beta dX R^T
    a = values(6)
    x["beta"][0], x["beta"][1], x["beta"][2] = 1, a, coarse(a)
    x["v"][0, ..., 0] = 1
    x["k"][0, ..., 0] = 1
    x["k"][1:, ..., 2] = 0.5
    x["k"][1, ..., 1], x["k"][2, ..., 1] = 0.5, -0.5
    gs[..., 2, 0] = 2
    return "grad_k", (0, ..., 1)


def rate_in_grad_v(x, go, gs):             # dV = beta dX with dX = K dS'
    a = values(7)
    gs[..., 0, 0], gs[..., 1, 0] = a, coarse(a)
    x["k"][0, ..., 0], x["k"][0, ..., 1] = 0.5, -0.5
    x["beta"][0] = 1
    return "grad_v", (0, ..., 0)


def rows_in_state(x, go, gs):              # S' = K^T R
    a = values(8)
    x["beta"][0], x["beta"][1] = a, coarse(a)
    x["v"][..., 0] = 1
    orthogonal_keys(x)
    return "last", (..., 0, 0)


def decay_in_state(x, go, gs):             # S' = K^T (d R) with d = e^g
    a = values(9)
    x["g"][1] = a.log()
    x["beta"][0], x["beta"][1] = 1, coarse(a)
    x["v"][..., 0] = 1
    orthogonal_keys(x)
    return "last", (..., 0, 0)


def decay_in_grad_state(x, go, gs):        # dS = Q^T (a dO)
    a = values(10)
    x["g"][0], x["g"][1] = a.log(), -2.0 ** -12
    x["q"][0, ..., 0], x["q"][1, ..., 0] = 1, -1
    go[..., 0] = 1
    return "grad_state", (..., 0, 0)


def products_in_grad_beta(x, go, gs):      # dbeta = v . dX with dX = K dS'
    a = values(11)
    gs[..., 0, 0], gs[..., 0, 1] = a, coarse(a)
    x["k"][0, ..., 0] = 1
    x["v"][0, ..., 0], x["v"][0, ..., 1] = 1, -1
    return "grad_beta", (0,)


def state_in_grad_g(x, go, gs):            # dg = a q . (S dO)
    a = values(12)
    x["state"][..., 0, 0], x["state"][..., 0, 1] = a, coarse(a)
    x["q"][0, ..., 0] = 1
    go[0, ..., 0], go[0, ..., 1] = 1, -1
    return "grad_g", (0,)


CASES = [state_in_output, rows_in_output, decay_in_output, scores_in_grad_q, state_in_grad_q, scores_in_grad_k,
         corrections_in_grad_k, rate_in_grad_v, rows_in_state, decay_in_state, decay_in_grad_state,
         products_in_grad_beta, state_in_grad_g]

def built(case):
    x, go, gs = blank()
    name, at = case(x, go, gs)
    return x, go, gs, name, at


def expected(x, go, gs, name):
    leaf = {n: t.double().requires_grad_(True) for n, t in x.items()}
    o, last = recurrence(leaf, None, 1.0)
    if not name.startswith("grad"):
        return {"o": o, "last": last}[name].detach()
    return torch.autograd.grad((o * go.double()).sum() + (last * gs.double()).sum(), leaf[name[5:]])[0]


def within(got, want):
    half = torch.finfo(got.dtype).eps / 2
    got = got.cpu().double()
    assert bool(torch.isfinite(got).all())
    over = (got - want).abs() - (BOUND + half * want.abs())
    assert bool((over <= 0).all()), f"off by up to {float((got - want).abs().max()):.3g}, allowed about {BOUND:.3g}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: c.__name__)
def test_differences_of_nearly_equal_terms(sf, case, dtype):
    x, go, gs, name, at = built(case)
    want = expected(x, go, gs, name)
    leaf = {n: (t.to(dtype) if n in "qkv" else t).cuda().requires_grad_(True) for n, t in x.items()}
    for n in "qkv":
        assert torch.equal(leaf[n].detach().cpu().float(), x[n])
    o, last = sf.gated_delta_func(*(leaf[n] for n in NAMES), None, 1.0)
    if name.startswith("grad"):
        got, = torch.autograd.grad((o, last), leaf[name[5:]], (go.to(dtype).cuda(), gs.cuda()))
    else:
        got = {"o": o, "last": last}[name].detach()
        with torch.no_grad():      # the form that leaves nothing for a backward
            plain = sf.gated_delta_func(*(leaf[n] for n in NAMES), None, 1.0)
        within(plain[0 if name == "o" else 1][at], want[at])
    within(got[at], want[at])
