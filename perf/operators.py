"""What the token layers cost: embedding, group norm with an activation, and the gated delta rule.

Each case is one call of a user's program.  ``run`` computes it either in its plain form -- elementary
torch operations in 32 bits, rounded once at the end -- or, where ``own`` is true, through the
framework's entry points; both start from what ``prepare`` returns.  ``exact`` is the operator's
definition in 64 bits.

Tensors are time-major, ``[T, B, ...]``, as everywhere in this repository.
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- cases --------------------------------------------------------------------------------------------------


def _embed(name, T, B, V, C, dtype, train, pad=False):
    return {"name": name, "op": "embed", "T": T, "B": B, "V": V, "C": C, "dtype": dtype, "train": train,
            "pad": pad}


def _gn(name, T, B, H, W, G, cpg, act, dtype, train):
    return {"name": name, "op": "gn", "T": T, "B": B, "H": H, "W": W, "G": G, "cpg": cpg, "act": act,
            "dtype": dtype, "train": train}


def _delta(name, T, B, Hk, Hv, Dk, Dv, dtype, mode, ragged=False, state=False):
    return {"name": name, "op": "delta", "T": T, "B": B, "Hk": Hk, "Hv": Hv, "Dk": Dk, "Dv": Dv,
            "dtype": dtype, "mode": mode, "ragged": ragged, "state": state}


def listed():
    return [
        # the input layer of one generated token for each of 64 sequences: pure latency
        _embed("embed_decode", 1, 64, 32000, 1024, "bf16", False),
        # a training batch of 32768 tokens over a 50000-word vocabulary, frequencies as in text
        _embed("embed_train", 2048, 16, 50000, 1024, "bf16", True),
        # a short ragged batch, odd in every size, in single precision; absent tokens are -1
        _embed("embed_train_odd", 333, 5, 5003, 250, "f32", True, pad=True),
        # the normalisation of one generated token for each of 32 sequences
        _gn("gn_decode", 1, 32, 1, 1, 8, 64, "silu", "bf16", False),
        # the activations of the benchmark's [8,64,128,32,32] layer with the channels innermost, a training step
        _gn("gn_train_images", 8, 64, 32, 32, 32, 4, "silu", "f32", True),
        # per-head normalisation of a token layer's output in a training step: 8 heads of 128 channels
        _gn("gn_train_tokens", 2048, 8, 1, 1, 8, 128, "silu", "bf16", True),
        # odd planes and groups
        _gn("gn_train_odd", 5, 7, 13, 11, 9, 10, "gelu", "f32", True),
        # one generated token for each of 64 sequences: the whole state is read and written
        _delta("delta_step", 1, 64, 8, 16, 128, 128, "bf16", "step"),
        # one token of one sequence: latency
        _delta("delta_step_single", 1, 1, 4, 4, 64, 64, "f32", "step"),
        # a long prompt of one sequence before generation: few heads, long chain
        _delta("delta_prefill", 8192, 1, 8, 16, 128, 128, "bf16", "forward", state=True),
        # a training step of one layer
        _delta("delta_train", 2048, 4, 8, 8, 128, 128, "bf16", "train"),
        # ragged batch, shared key heads, odd sizes, single precision, a state carried in
        _delta("delta_train_odd", 777, 3, 2, 4, 96, 80, "f32", "train", ragged=True, state=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "gn", "delta", "delta"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "embed":
        train = rng.random() < 0.7
        C = _log_int(rng, 8, 2048)
        V = _log_int(rng, 10, 60000)
        while V * C > 50000 * 1024:
            V = _log_int(rng, 10, 60000)
        n_max = min(65536, 2048 * 16 * 1024 // C)
        n = _log_int(rng, 1, n_max)
        B = _log_int(rng, 1, min(64, n))
        if dtype == "f32":            # twice the bytes
            C = max(4, C // 2)
        return _embed(None, max(1, n // B), B, V, C, dtype, train, pad=rng.random() < 0.5)
    if op == "gn":
        G = rng.choice([1, 2, 3, 4, 8, 9, 16, 32])
        cpg = _log_int(rng, 1, 128)
        side = rng.choice([(1, 1), (1, 1), (rng.randint(2, 64), rng.randint(2, 64))])
        per = G * cpg * side[0] * side[1]
        samples = _log_int(rng, 1, max(1, min(16384, 8 * 64 * 128 * 1024 // (2 * per))))
        B = _log_int(rng, 1, min(64, samples))
        return _gn(None, max(1, samples // B), B, side[0], side[1], G, cpg,
                   rng.choice(["none", "relu", "silu", "gelu"]), dtype, rng.random() < 0.7)
    mode = rng.choice(["train", "train", "forward", "step"])
    Hk = rng.choice([1, 2, 3, 4, 8])
    Hv = Hk * rng.choice([1, 1, 2, 4])
    Dk = rng.choice([16, 32, 64, 64, 96, 128, 128, rng.randint(16, 128)])
    Dv = rng.choice([16, 32, 64, 64, 96, 128, 128, rng.randint(16, 128)])
    if mode == "step":
        return _delta(None, 1, _log_int(rng, 1, 64 * 16 // Hv), Hk, Hv, Dk, Dv, dtype, mode)
    # no more than the listed training step (2048 x 4 x 8 heads) or, forward only, the listed prompt
    total = 2048 * 4 * 8 if mode == "train" else 8192 * 16
    if dtype == "f32":
        total //= 2
    T = _log_int(rng, 1, 2048 if mode == "train" else 8192)
    T = min(T, total // Hv)
    B = _log_int(rng, 1, max(1, min(16, total // (T * Hv))))
    return _delta(None, T, B, Hk, Hv, Dk, Dv, dtype, mode, ragged=rng.random() < 0.3, state=rng.random() < 0.5)


# ---- inputs -------------------------------------------------------------------------------------------------


def _generator(seed, salt):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1000003 * int(seed) + salt)
    return gen


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _rand(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda")


def prepare(case, seed):
    dt = _DTYPES[case["dtype"]]
    T, B = case["T"], case["B"]
    s = {"case": case}
    if case["op"] == "embed":
        gen = _generator(seed, 1)
        V, C = case["V"], case["C"]
        # word frequencies fall as 1 / rank; ranks lie anywhere in the table
        rank = torch.exp(_rand(gen, T, B) * math.log(V + 1)).long().sub_(1).clamp_(0, V - 1)
        tokens = torch.randperm(V, generator=gen, device="cuda")[rank]
        if case["pad"]:           # a sequence ends anywhere in its second half
            ends = (T * (0.5 + 0.5 * _rand(gen, B))).long()
            tokens = torch.where(torch.arange(T, device="cuda")[:, None] > ends, -1, tokens)
        s.update(tokens=tokens, weight=(_randn(gen, V, C) / math.sqrt(C)).to(dt), scale=math.sqrt(C))
        if case["train"]:
            s["weight"].requires_grad_(True)
            s["grad"] = _randn(gen, T, B, C).to(dt)
    elif case["op"] == "gn":
        gen = _generator(seed, 2)
        C = case["G"] * case["cpg"]
        shape = (T, B, C) if case["H"] * case["W"] == 1 else (T, B, case["H"], case["W"], C)
        spread = 0.5 + _rand(gen, C)
        s.update(x=(_randn(gen, *shape) * spread + 0.5 * _randn(gen, C)).to(dt),
                 weight=(0.5 + _rand(gen, C)).to(dt), bias=(0.2 * _randn(gen, C)).to(dt))
        if case["train"]:
            s["grad"] = _randn(gen, *shape).to(dt)
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_(True)
    else:
        gen = _generator(seed, 3)
        Hk, Hv, Dk, Dv = case["Hk"], case["Hv"], case["Dk"], case["Dv"]
        unit = lambda x: x / x.norm(dim=-1, keepdim=True)
        # decays from nearly one (long memory) to about a half, another rate for each head
        rate = torch.exp(torch.linspace(math.log(0.005), math.log(0.5), Hv, device="cuda"))
        s.update(q=unit(_randn(gen, T, B, Hk, Dk)).to(dt), k=unit(_randn(gen, T, B, Hk, Dk)).to(dt),
                 v=_randn(gen, T, B, Hv, Dv).to(dt),
                 g=-rate * torch.nn.functional.softplus(_randn(gen, T, B, Hv)),
                 beta=torch.sigmoid(_randn(gen, T, B, Hv)),
                 state=None, lengths=None, scale=Dk ** -0.5)
        if case["state"] or case["mode"] == "step":
            s["state"] = 0.3 * _randn(gen, B, Hv, Dk, Dv)
        if case["mode"] == "step":
            s["state_out"] = torch.empty_like(s["state"])
        if case["ragged"]:
            s["lengths"] = (T * (0.3 + 0.7 * _rand(gen, B))).ceil().to(torch.int32).clamp_(0, T)
        if case["mode"] == "train":
            s["grad"] = _randn(gen, T, B, Hv, Dv).to(dt)
            s["grad_state"] = 0.1 * _randn(gen, B, Hv, Dk, Dv)
            for name in ("q", "k", "v", "g", "beta") + (("state",) if case["state"] else ()):
                s[name].requires_grad_(True)
    return s


# ---- the framework's calls ----------------------------------------------------------------------------------


def _run_own(s):
    from snn_gpu_training_bptt_amd import snnlib_func as sf
    case = s["case"]
    if case["op"] == "embed":
        if not case["train"]:
            return sf.embed_func(s["tokens"], s["weight"], s["scale"])
        y = sf.embed_func(s["tokens"], s["weight"], s["scale"])
        return (y.detach(),) + torch.autograd.grad(y, (s["weight"],), s["grad"])
    if case["op"] == "gn":
        y = sf.gn_act_func(s["x"], s["weight"], s["bias"], case["G"], 1e-5, case["act"])
        if not case["train"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])
    if case["mode"] == "step":
        o = sf.gated_delta_step(s["q"][0], s["k"][0], s["v"][0], s["g"][0], s["beta"][0], s["state"], s["scale"],
                                s["state_out"])
        return o, s["state_out"]
    o, last = sf.gated_delta_func(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["lengths"], s["scale"])
    if case["mode"] == "forward":
        return o, last
    leaves = [s[n] for n in ("q", "k", "v", "g", "beta")] + ([s["state"]] if case["state"] else [])
    grads = torch.autograd.grad((o, last), leaves, (s["grad"], s["grad_state"]))
    return (o.detach(), last.detach()) + grads


# ---- the plain form -----------------------------------------------------------------------------------------


def _act_plain(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _gn_plain(x, weight, bias, G, act):
    T, B, C = x.shape[0], x.shape[1], x.shape[-1]
    xg = x.float().reshape(T * B, -1, G, C // G)
    mean = xg.mean(dim=(1, 3), keepdim=True)
    centred = xg - mean
    var = (centred * centred).mean(dim=(1, 3), keepdim=True)
    z = (centred / torch.sqrt(var + 1e-5)).reshape(x.shape) * weight.float() + bias.float()
    return _act_plain(z, act)


def _delta_plain(q, k, v, g, beta, state, lengths, scale):
    """The recurrence as it is defined, one time step after the other."""
    T, B, Hv, Dv = v.shape
    times = Hv // k.shape[2]
    q, k = (t.float().repeat_interleave(times, dim=2) for t in (q, k))
    v, alpha = v.float(), torch.exp(g)
    if lengths is not None:
        there = (torch.arange(T, device=v.device)[:, None] < lengths[None, :])[..., None]
        alpha = torch.where(there, alpha, 1.0)
        beta = torch.where(there, beta, 0.0)
        q = q * there[..., None]
    S = state if state is not None else v.new_zeros(B, Hv, k.shape[-1], Dv)
    out = []
    for t in range(T):
        S = S * alpha[t][..., None, None]
        kt = k[t][..., None, :]                                     # [B, H, 1, Dk]
        error = beta[t][..., None, None] * (v[t][..., None, :] - torch.matmul(kt, S))
        S = S + kt.transpose(-1, -2) * error
        out.append(torch.matmul(q[t][..., None, :], S)[..., 0, :])
    return torch.stack(out) * scale, S


def _run_plain(s):
    case = s["case"]
    dt = _DTYPES[case["dtype"]]
    if case["op"] == "embed":
        tokens, weight = s["tokens"], s["weight"].detach()
        there = (tokens >= 0) & (tokens < weight.shape[0])
        rows = torch.where(there, tokens, 0).reshape(-1)
        y = weight[rows].float() * s["scale"] * there.reshape(-1, 1)
        y = y.to(dt).reshape(*tokens.shape, -1)
        if not case["train"]:
            return y
        g = s["grad"].float().reshape(-1, weight.shape[1]) * there.reshape(-1, 1)
        grad = torch.zeros(weight.shape, device=g.device).index_add_(0, rows, g) * s["scale"]
        return y, grad.to(dt)
    if case["op"] == "gn":
        y = _gn_plain(s["x"], s["weight"], s["bias"], case["G"], case["act"])
        if not case["train"]:
            return y.to(dt)
        leaves = (s["x"], s["weight"], s["bias"])
        return (y.detach().to(dt),) + torch.autograd.grad(y, leaves, s["grad"].float())
    args = [s[n] for n in ("q", "k", "v", "g", "beta", "state", "lengths", "scale")]
    if case["mode"] != "train":
        with torch.no_grad():
            o, last = _delta_plain(*args)
        return (o[0] if case["mode"] == "step" else o).to(dt), last
    o, last = _delta_plain(*args)
    leaves = [s[n] for n in ("q", "k", "v", "g", "beta")] + ([s["state"]] if case["state"] else [])
    grads = torch.autograd.grad((o, last), leaves, (s["grad"].float(), s["grad_state"]))
    return (o.detach().to(dt), last.detach()) + grads


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits ------------------------------------------------------------------------------


def _embed_exact(s):
    case = s["case"]
    tokens = s["tokens"].reshape(-1).cpu().numpy()
    weight = s["weight"].detach().double().cpu().numpy()
    V, C = weight.shape
    there = (tokens >= 0) & (tokens < V)
    y = np.zeros((tokens.size, C))
    y[there] = weight[tokens[there]] * s["scale"]
    y = torch.from_numpy(y.reshape(case["T"], case["B"], C))
    if not case["train"]:
        return y
    g = s["grad"].double().reshape(-1, C).cpu().numpy()
    order = np.argsort(tokens, kind="stable")
    order = order[there[order]]
    grad = np.zeros((V, C))
    if order.size:
        sorted_tokens = tokens[order]
        first = np.flatnonzero(np.r_[True, sorted_tokens[1:] != sorted_tokens[:-1]])
        grad[sorted_tokens[first]] = np.add.reduceat(g[order], first, axis=0) * s["scale"]
    return y, torch.from_numpy(grad)


def _gn_exact(s):
    case = s["case"]
    G = case["G"]
    x = s["x"].detach().double()
    shape, C = x.shape, x.shape[-1]
    x = x.reshape(shape[0] * shape[1], -1, G, C // G)
    w = s["weight"].detach().double().reshape(1, 1, G, -1)
    b = s["bias"].detach().double().reshape(1, 1, G, -1)
    var, mean = torch.var_mean(x, dim=(1, 3), keepdim=True, unbiased=False)
    inv = (var + 1e-5).rsqrt()
    xhat = (x - mean) * inv
    z = torch.addcmul(b, xhat, w)
    act = case["act"]
    if act == "relu":
        y, slope = torch.relu(z), (z > 0).double()
    elif act == "silu":
        sig = torch.sigmoid(z)
        y, slope = z * sig, sig * (1 + z * (1 - sig))
    elif act == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        y, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    else:
        y, slope = z, torch.ones_like(z)
    if not case["train"]:
        return y.reshape(shape)
    gz = s["grad"].double().reshape(x.shape) * slope
    grad_w, grad_b = (gz * xhat).sum(dim=(0, 1)).reshape(C), gz.sum(dim=(0, 1)).reshape(C)
    gx = gz * w
    gx = inv * (gx - gx.mean(dim=(1, 3), keepdim=True) - xhat * (gx * xhat).mean(dim=(1, 3), keepdim=True))
    return y.reshape(shape), gx.reshape(shape), grad_w, grad_b


def _delta_exact(s):
    """Chunks of 32 steps, each a triangular system, in 64 bits on the CPU; gradients by differentiating that."""
    case = s["case"]
    names = ["q", "k", "v", "g", "beta"] + (["state"] if s["state"] is not None else [])
    leaf = {n: s[n].detach().double().cpu().requires_grad_(case["mode"] == "train") for n in names}
    T, B, Hv, Dk, Dv = case["T"], case["B"], case["Hv"], case["Dk"], case["Dv"]
    times = Hv // case["Hk"]

    def heads_first(x, reps=1):                              # [T, B, H, ...] -> [B, H, T, ...]
        x = x.movedim(0, 2)
        return x.repeat_interleave(reps, dim=1) if reps > 1 else x

    q, k = heads_first(leaf["q"], times), heads_first(leaf["k"], times)
    v, g, beta = (heads_first(leaf[n]) for n in ("v", "g", "beta"))
    if s["lengths"] is not None:
        there = torch.arange(T)[None, None, :] < s["lengths"].cpu().long()[:, None, None]
        g, beta = g * there, beta * there
        q = q * there[..., None]
    S = leaf.get("state", torch.zeros(B, Hv, Dk, Dv, dtype=torch.double))
    out = []
    for t0 in range(0, T, 32):
        qc, kc, vc = (x[:, :, t0:t0 + 32] for x in (q, k, v))
        bc = beta[:, :, t0:t0 + 32, None]
        total = g[:, :, t0:t0 + 32].cumsum(-1)
        n = total.shape[-1]
        lower = torch.ones(n, n, dtype=torch.bool).tril()
        decay = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill(~lower, -math.inf))
        system = torch.eye(n, dtype=torch.double) + (bc * (kc @ kc.mT) * decay).tril(-1)
        new = torch.linalg.solve_triangular(system, bc * (vc - total.exp()[..., None] * (kc @ S)),
                                            upper=False, unitriangular=True)
        out.append(total.exp()[..., None] * (qc @ S) + ((qc @ kc.mT) * decay) @ new)
        rest = torch.exp(total[..., -1:] - total)[..., None]
        S = total[..., -1].exp()[..., None, None] * S + (rest * kc).mT @ new
    o = torch.cat(out, dim=2).movedim(2, 0) * s["scale"]
    if case["mode"] == "step":
        return o[0], S
    if case["mode"] == "forward":
        return o, S
    grads = torch.autograd.grad((o, S), [leaf[n] for n in names],
                                (s["grad"].double().cpu(), s["grad_state"].double().cpu()))
    return (o.detach(), S.detach()) + grads


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        return _embed_exact(s)
    return _gn_exact(s) if case["op"] == "gn" else _delta_exact(s)


# ---- what a pass cannot do without --------------------------------------------------------------------------


def work(case):
    size = _DTYPES[case["dtype"]].itemsize
    T, B = case["T"], case["B"]
    if case["op"] == "embed":
        n, C, V = T * B, case["C"], case["V"]
        rows = min(n, V)                                 # distinct rows read, at most
        nbytes = 8 * n + size * C * (rows + n)
        flops = n * C
        if case["train"]:
            nbytes += size * C * (n + V)
            flops += 2 * n * C
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "gn":
        n = T * B * case["H"] * case["W"] * case["G"] * case["cpg"]
        return {"bytes": size * n * (5 if case["train"] else 2), "flops": n * (30 if case["train"] else 10)}
    Hk, Hv, Dk, Dv = case["Hk"], case["Hv"], case["Dk"], case["Dv"]
    qkvo = T * B * (2 * Hk * Dk + 2 * Hv * Dv) * size + 8 * T * B * Hv
    state = 4 * B * Hv * Dk * Dv
    states = (2 if case["state"] or case["mode"] == "step" else 1) * state
    flops = 7 * T * B * Hv * Dk * Dv
    if case["mode"] == "train":      # the gradients in, the inputs once more, their gradients out
        return {"bytes": 2 * qkvo + T * B * (2 * Hk * Dk + Hv * Dv) * size + 8 * T * B * Hv + 2 * states,
                "flops": 3 * flops}
    return {"bytes": qkvo + states, "flops": flops}


if __name__ == "__main__":
    for case in listed() + [draw(random.Random(i)) for i in range(4)]:
        print(case, work(case))
