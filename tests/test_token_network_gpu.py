"""The token layers together, as a network over sequences uses them: embedding, group norm, projections to queries, keys,
values and gates, the gated delta rule, a norm per head, the read-out; trained through time on a ragged batch, and
generating token by token."""
import math

import pytest
import torch

from snn_gpu_training_bptt_amd import lif_cabi  # noqa: F401

pytestmark = pytest.mark.gpu
V, C, HK, HV, DK, DV = 37, 48, 2, 4, 16, 24
SPLIT = [HK * DK, HK * DK, HV * DV, HV, HV]


def network(seed=0):
    """One block on the framework's layers: ``Embed -> GnAct -> Fc -> GatedDelta -> GnAct -> Fc``."""
    from snn_gpu_training_bptt_amd import snnlib_op as sop

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.embed = sop.Embed(V, C, math.sqrt(C))
            self.norm = sop.GnAct(4, C, act="gelu")
            self.project = sop.Fc(C, sum(SPLIT))
            self.delta = sop.GatedDelta()
            self.head_norm = sop.GnAct(HV, HV * DV, act="silu")
            self.read = sop.Fc(HV * DV, V)

        def operands(self, tokens):
            T, B = tokens.shape
            p = self.project(self.norm(self.embed(tokens))).split(SPLIT, dim=-1)
            unit = lambda x: torch.nn.functional.normalize(x.reshape(T, B, HK, DK), dim=-1)
            return (unit(p[0]), unit(p[1]), p[2].reshape(T, B, HV, DV), -torch.nn.functional.softplus(p[3]),
                    torch.sigmoid(p[4]))

        def forward(self, tokens, lengths=None, state=None):
            o, state = self.delta(*self.operands(tokens), state, lengths)
            return self.read(self.head_norm(o.flatten(2))), state

        def generate(self, token, state):
            q, k, v, g, beta = (t[0] for t in self.operands(token[None]))
            o = self.delta.step(q, k, v, g, beta, state)
            return self.read(self.head_norm(o.flatten(1)[None]))[0]

    torch.manual_seed(seed)
    return Net().cuda()


def plain(params, tokens, lengths):
    """The same network in 64 bits on the host, from elementary operations."""
    T, B = tokens.shape
    there = tokens >= 0
    x = params["embed.weight_embed"][tokens.clamp_min(0)] * math.sqrt(C) * there[..., None]

    def norm(x, groups, w, b):
        y = x.reshape(T, B, groups, -1)
        y = y - y.mean(-1, keepdim=True)
        return (y / (y.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()).reshape(x.shape) * w + b

    h = norm(x, 4, params["norm.weight_gn"], params["norm.bias_gn"])
    h = 0.5 * h * (1 + torch.erf(h / math.sqrt(2)))
    p = (h @ params["project.weight_fc"].T + params["project.bias_fc"]).split(SPLIT, dim=-1)
    heads = lambda x, n: x.reshape(T, B, n, -1)
    # rows of absent tokens have projections of zero: torch's normalize divides those by 1e-12
    unit = lambda x: x / x.norm(dim=-1, keepdim=True).clamp_min(1e-12)
    q, k = (unit(heads(t, HK)).repeat_interleave(HV // HK, dim=2) for t in p[:2])
    v, g, beta = heads(p[2], HV), -torch.log1p(torch.exp(p[3])), 1 / (1 + torch.exp(-p[4]))
    S, out = torch.zeros(B, HV, DK, DV, dtype=torch.float64), []
    for t in range(T):
        m = (t < lengths)[:, None, None, None]
        decayed = torch.exp(g[t])[..., None, None] * S
        error = beta[t][..., None] * (v[t] - (decayed * k[t][..., None]).sum(-2))
        S = torch.where(m, decayed + k[t][..., None] * error[..., None, :], S)
        out.append(torch.where(m[..., 0], (S * q[t][..., None]).sum(-2) * DK ** -0.5, 0.0))
    o = norm(torch.stack(out).flatten(2), HV, params["head_norm.weight_gn"], params["head_norm.bias_gn"])
    return (o / (1 + torch.exp(-o))) @ params["read.weight_fc"].T + params["read.bias_fc"]


def batch(T=70, B=3, seed=1):
    gen = torch.Generator().manual_seed(seed)
    lengths = torch.tensor([T, 41, 65][:B], dtype=torch.int32)
    tokens = torch.randint(0, V, (T, B), generator=gen)
    there = torch.arange(T)[:, None] < lengths
    return torch.where(there, tokens, -1), torch.randint(0, V, (T, B), generator=gen), lengths, there


def loss_of(logits, labels, there):
    each = torch.nn.functional.cross_entropy(logits.flatten(0, 1), labels.flatten(), reduction="none")
    return (each * there.flatten()).sum() / there.sum()


def test_gradients_of_a_training_step():
    """Against 64 bits.  Every layer and library product is good to about 2**-20 of its norm (sums of up to a hundred fp32
    products); a gradient passes some 30 of them, and the group norms divide by a spread that is below one: within
    2**-20 * 30 * 8 < 3e-4 of the largest value of each parameter's gradient."""
    net = network()
    tokens, labels, lengths, there = batch()
    logits, _ = net(tokens.cuda(), lengths.cuda())
    loss = loss_of(logits, labels.cuda(), there.cuda())
    loss.backward()
    params = {n: p.detach().cpu().double().requires_grad_(True) for n, p in net.named_parameters()}
    want = plain(params, tokens, lengths)
    want_loss = loss_of(want, labels, there)
    want_loss.backward()
    want, want_loss = want.detach(), want_loss.detach()
    valid = there[..., None].expand_as(want)
    assert float((logits.detach().cpu().double() - want)[valid].abs().max()) <= 3e-4 * float(want.abs().max())
    assert abs(float(loss.detach()) - float(want_loss)) <= 3e-4 * float(want_loss)
    for n, p in net.named_parameters():
        e = params[n].grad
        assert float((p.grad.cpu().double() - e).abs().max()) <= 3e-4 * float(e.abs().max()), n


def test_what_lies_behind_the_lengths_does_not_matter():
    net = network()
    tokens, labels, lengths, there = batch()
    grads = []
    for fill in (-1, 5):
        net.zero_grad()
        logits, last = net(torch.where(there, tokens, fill).cuda(), lengths.cuda())
        loss_of(logits, labels.cuda(), there.cuda()).backward()
        grads.append([last.detach()] + [p.grad.clone() for p in net.parameters()])
    for a, b in zip(*grads):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6 * float(b.abs().max()))


def test_generation_continues_a_prompt():
    """A prompt through the chunked form, then one token at a time, against the whole sequence at once."""
    net = network()
    gen = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, V, (80, 2), generator=gen).cuda()
    with torch.no_grad():
        whole, whole_state = net(tokens)
        prompt, state = net(tokens[:67])
        rest = torch.stack([net.generate(tokens[t], state) for t in range(67, 80)])
    torch.testing.assert_close(prompt, whole[:67], rtol=1e-4, atol=1e-4 * float(whole.abs().max()))
    torch.testing.assert_close(rest, whole[67:], rtol=1e-4, atol=1e-4 * float(whole.abs().max()))
    torch.testing.assert_close(state, whole_state, rtol=1e-4, atol=1e-4 * float(whole_state.abs().max()))


def test_a_training_step_is_captured_and_replayed():
    """Forward, backward and update in one graph, replayed with new tokens, against the same steps run eagerly."""
    tokens, labels, lengths, there = batch()
    gen = torch.Generator().manual_seed(9)
    fresh = [torch.where(there, torch.randint(0, V, tokens.shape, generator=gen), -1).cuda() for _ in range(4)]
    labels, lengths, there = labels.cuda(), lengths.cuda(), there.cuda()

    def step(net, tokens):
        logits, _ = net(tokens, lengths)
        grads = torch.autograd.grad(loss_of(logits, labels, there), list(net.parameters()))
        with torch.no_grad():
            for p, g in zip(net.parameters(), grads):
                p.sub_(0.1 * g)
        return grads

    eager, captured = network(5), network(5)
    x = tokens.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(captured, x)                        # warm up, off the capturing stream
    torch.cuda.current_stream().wait_stream(side)
    captured.load_state_dict(eager.state_dict())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured, x)
    captured.load_state_dict(eager.state_dict())
    for t in fresh:
        x.copy_(t)
        graph.replay()
        step(eager, t)
        torch.cuda.synchronize()
        for (n, a), b in zip(captured.named_parameters(), eager.parameters()):
            torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5, msg=lambda m: f"{n}: {m}")
