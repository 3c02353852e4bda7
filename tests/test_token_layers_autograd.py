"""What autograd and graph tracers must not get from the token layers in silence: every entry either takes part or refuses."""
import pytest
import torch
from torch.autograd import forward_ad

from snn_gpu_training_bptt_amd import lif_cabi  # noqa: F401  (fails loudly without the built library)
from snn_gpu_training_bptt_amd import snnlib_func as sf

devices = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


def operands(device):
    """Per entry: the call, and its floating operands by name."""
    gen = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=gen).to(device)
    tokens = torch.randint(0, 5, (3, 2), generator=gen).to(device)
    rule = dict(q=rand(3, 2, 1, 4), k=0.3 * rand(3, 2, 1, 4), v=rand(3, 2, 1, 4), g=-rand(3, 2, 1).abs(),
                beta=rand(3, 2, 1).sigmoid(), state=rand(2, 1, 4, 4))
    row = {n: t if n == "state" else t[0] for n, t in rule.items()}
    norm = dict(x=rand(3, 2, 4), weight=rand(4), bias=rand(4))
    six = lambda a: [a[n] for n in ("q", "k", "v", "g", "beta", "state")]
    return {
        "embed": (lambda a: sf.embed_func(tokens, a["weight"]), dict(weight=rand(5, 4))),
        "embed_fp": (lambda a: sf.snnlib.embed_fp(tokens, a["weight"], 1.0), dict(weight=rand(5, 4))),
        "embed_bp": (lambda a: sf.snnlib.embed_bp(tokens, a["grad"], 5, 1.0), dict(grad=rand(3, 2, 4))),
        "gn_act": (lambda a: sf.gn_act_func(a["x"], a["weight"], a["bias"], 2), norm),
        "gn_act_fp": (lambda a: sf.snnlib.gn_act_fp(a["x"], a["weight"], a["bias"], 2, 1e-5, "silu"), norm),
        "gn_act_bp": (lambda a: sf.snnlib.gn_act_bp(a["x"], a["weight"], a["bias"], a["mean"], a["rstd"], 2, "silu", a["grad"]),
                      dict(norm, mean=rand(3, 2, 2), rstd=rand(3, 2, 2).abs(), grad=rand(3, 2, 4))),
        "gated_delta": (lambda a: sf.gated_delta_func(*six(a)), rule),
        "gated_delta_fp": (lambda a: sf.snnlib.gated_delta_fp(*six(a), None, 1.0), rule),
        "gated_delta_bp": (lambda a: sf.snnlib.gated_delta_bp(*six(a), None, 1.0, torch.empty(0, dtype=torch.uint8, device=device),
                                                              a["grad"], a["grad_state"]),
                           dict(rule, grad=rand(3, 2, 1, 4), grad_state=rand(2, 1, 4, 4))),
        "gated_delta_step": (lambda a: sf.gated_delta_step(*six(a), None, a["state_out"]), dict(row, state_out=rand(2, 1, 4, 4))),
    }


ENTRIES = list(operands("cpu"))


@devices
@pytest.mark.parametrize("entry", ENTRIES)
def test_forward_mode_is_refused(entry, device):
    """A tangent on any operand, with and without gradients: an error, never an output without a tangent."""
    call, args = operands(device)[entry]
    for name in args:
        for grad in (False, True):
            with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                dual = dict(args)
                primal = args[name].clone().requires_grad_(grad and entry in ("embed", "gn_act", "gated_delta"))
                dual[name] = forward_ad.make_dual(primal, torch.ones_like(primal))
                with pytest.raises((RuntimeError, NotImplementedError), match="forward-mode|Jacobian-vector product"):
                    call(dual)


@pytest.mark.gpu
@pytest.mark.parametrize("entry", ["embed", "gn_act", "gated_delta"])
def test_forward_mode_through_a_backward_is_refused(entry):
    call, args = operands("cuda")[entry]
    leaf = {n: t.requires_grad_(True) for n, t in args.items()}
    y = call(leaf)
    y = y[0] if isinstance(y, tuple) else y
    with forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="forward-mode"):
            torch.autograd.grad(y, list(leaf.values()), forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)), allow_unused=True)


@devices
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("entry", ENTRIES)
def test_recording_a_graph_is_refused(entry, grad, device):
    """A tracer sees an output's allocation and not the kernel that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    call, args = operands(device)[entry]
    names = list(args)
    tracked = grad and entry in ("embed", "gn_act", "gated_delta")
    values = tuple(args[n].clone().requires_grad_(tracked) for n in names)
    run = lambda *t: call(dict(zip(names, t)))
    with pytest.raises(RuntimeError, match="cannot be recorded"):
        torch.jit.trace(run, values, check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be recorded"):
        make_fx(run)(*(t.detach() for t in values))


@pytest.mark.parametrize("entry", ENTRIES)
def test_fake_tensors_are_refused(entry):
    """They are on a GPU by name, and their address is their offset: nothing a kernel may follow."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True):
        call, args = operands("cuda")[entry]
        for offset in (0, 3):
            views = {}
            for n, t in args.items():
                wide = torch.empty(t.numel() + offset, device="cuda")
                views[n] = wide[offset:].view(t.shape)
            with pytest.raises(RuntimeError, match="has no memory"):
                call(views)


@pytest.mark.gpu
@pytest.mark.parametrize("entry", ENTRIES)
def test_one_fake_tensor_among_others_is_refused(entry):
    from torch._subclasses.fake_tensor import FakeTensorMode
    call, args = operands("cuda")[entry]
    for name in args:
        mode = FakeTensorMode()
        fake = mode.from_tensor(torch.empty(args[name].numel() + 3, device="cuda"))
        with mode:
            fake = fake[3:].view(args[name].shape)
        with pytest.raises(RuntimeError, match="has no memory|what gated_delta_fp returned"):
            call({**args, name: fake})


@pytest.mark.gpu
@pytest.mark.parametrize("entry", ["embed", "gn_act", "gated_delta"])
def test_function_transforms_are_refused(entry):
    call, args = operands("cuda")[entry]
    names = list(args)

    def run(*t):
        y = call(dict(zip(names, t)))
        return (y[0] if isinstance(y, tuple) else y).sum()

    with pytest.raises(RuntimeError):
        torch.func.grad(run)(*args.values())
    with pytest.raises(RuntimeError):
        torch.func.jvp(run, tuple(args.values()), tuple(args.values()))
    with pytest.raises(RuntimeError):
        torch.func.vmap(run)(*(t.expand(2, *t.shape) for t in args.values()))


@devices
def test_a_step_into_a_tracked_state_is_refused(device):
    """state_out is overwritten: with gradients on, a parameter or a result with a history would keep what it no longer
    is the result of."""
    call, args = operands(device)["gated_delta_step"]
    leaf = args["state_out"].requires_grad_(True)
    for tracked in (leaf, leaf * 2):
        kept = tracked.detach().clone()
        with pytest.raises(RuntimeError, match="not differentiable"):
            call({**args, "state_out": tracked})
        assert torch.equal(tracked.detach(), kept)
    if device == "cuda":
        with torch.no_grad():
            call({**args, "state_out": leaf})
        assert not torch.equal(leaf.detach(), kept)


@devices
def test_keys_without_values_are_refused_as_such(device):
    """Also where the scale is left to its default, Dk ** -0.5."""
    q, g = torch.zeros(3, 2, 1, 0, device=device), torch.zeros(3, 2, 1, device=device)
    v, state = torch.zeros(3, 2, 1, 4, device=device), torch.zeros(2, 1, 0, 4, device=device)
    match = "ROCm GPU" if device == "cpu" else "keys of 1 to 128"
    with pytest.raises(RuntimeError, match=match):
        sf.gated_delta_func(q, q, v, g, g, state)
    with pytest.raises(RuntimeError, match=match):
        sf.gated_delta_step(q[0], q[0], v[0], g[0], g[0], state)
