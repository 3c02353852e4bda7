"""The token layers' boundary: the C ABI of include/snnlib_seq.h (symbols, constants, argument errors that need no GPU)
and the Python surface; on the GPU, the operators called through the C ABI alone."""
import ctypes
import os
import re

import pytest
import torch

from snn_gpu_training_bptt_amd import lif_cabi, seq_cabi

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(REPO, "include", "snnlib_seq.h")
F32, F64, BF16 = lif_cabi.DTYPE_F32, lif_cabi.DTYPE_F64, lif_cabi.DTYPE_BF16


def header_text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_header_table_and_library_agree():
    declared = sorted(set(re.findall(r"\b(snnseq_\w+)\s*\(", header_text())))
    assert declared == sorted(seq_cabi.SYMBOLS)
    lib = ctypes.CDLL(lif_cabi.LIB_PATH)
    for name in declared:
        assert hasattr(lib, name), f"{name} is declared but not exported"


def test_constants_match_the_header():
    macros = {k: int(v) for k, v in re.findall(r"#define\s+(SNNSEQ_\w+)\s+(\d+)", open(HEADER).read())}
    assert macros["SNNSEQ_ABI_VERSION"] == seq_cabi.ABI_VERSION == seq_cabi.load().snnseq_abi_version()
    assert (macros["SNNSEQ_TOKEN_I32"], macros["SNNSEQ_TOKEN_I64"]) == (seq_cabi.TOKEN_I32, seq_cabi.TOKEN_I64)
    assert {n: macros["SNNSEQ_ACT_" + n.upper()] for n in seq_cabi.ACTS} == seq_cabi.ACTS
    for name in ("TOKENS", "CHANNELS", "KEY", "VALUE", "HEADS"):
        assert macros["SNNSEQ_MAX_" + name] == getattr(seq_cabi, "MAX_" + name)


def test_argument_errors_need_no_gpu():
    """Stand-in pointers, aligned and never followed: every call here is refused, or has nothing to do."""
    lib = seq_cabi.load()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4098)
    fp = lambda dtype=F32, tok=1, N=4, V=5, C=6, t=p, w=p, o=p: lib.snnseq_embed_fp(t, w, o, dtype, tok, N, V, C, C, 1.0, None)
    assert fp(dtype=7) == seq_cabi.ERR_DTYPE and fp(tok=2) == seq_cabi.ERR_DTYPE
    assert fp(N=-1) == fp(V=0) == fp(C=-1) == fp(N=seq_cabi.MAX_TOKENS + 1) == seq_cabi.ERR_ARG
    assert fp(V=seq_cabi.MAX_TOKENS + 1) == fp(C=seq_cabi.MAX_CHANNELS + 1) == seq_cabi.ERR_ARG
    assert fp(t=None) == fp(w=None) == fp(o=None) == seq_cabi.ERR_ARG
    assert fp(w=odd) == fp(t=odd) == seq_cabi.ERR_ALIGN
    assert fp(N=0, t=None) == fp(C=0, t=None) == seq_cabi.OK
    need = lib.snnseq_embed_bp_workspace_bytes(F32, 100, 50, 8)
    assert need == 208 + 400 + 400 + 7 * 2 * 8 * 4             # start, positions, tokens, seven pieces' sums
    bp = lambda ws=p, n=need: lib.snnseq_embed_bp(p, p, p, F32, 1, 100, 50, 8, 1.0, ws, n, None)
    assert bp(n=need - 1) == bp(ws=None) == seq_cabi.ERR_WORKSPACE and bp(ws=odd) == seq_cabi.ERR_ALIGN
    assert lib.snnseq_embed_bp_workspace_bytes(F32, -1, 50, 8) == 0

    gn = lambda S=2, P=3, C=8, G=2, act=0, dtype=F32, x=p: lib.snnseq_gn_act_fp(x, p, p, p, p, p, dtype, S, P, C, G, 1e-5, act, None, 0, None)
    assert gn(dtype=9) == seq_cabi.ERR_DTYPE
    assert gn(G=3) == gn(G=0) == gn(S=-1) == gn(act=4) == gn(P=0) == gn(C=0) == gn(x=None) == seq_cabi.ERR_ARG
    assert gn(S=seq_cabi.MAX_TOKENS, G=2) == gn(P=seq_cabi.MAX_TOKENS + 1) == seq_cabi.ERR_ARG
    assert gn(S=0, P=0) == seq_cabi.OK and gn(x=odd) == seq_cabi.ERR_ALIGN
    assert lib.snnseq_gn_act_workspace_bytes(F32, 2, 3, 8, 2, 0) == 0
    assert lib.snnseq_gn_act_workspace_bytes(F32, 2, 3, 8, 2, 1) > 0
    assert lib.snnseq_gn_act_workspace_bytes(F32, 2, 3, 8, 3, 1) == 0
    assert lib.snnseq_gn_act_bp(*[p] * 9, F32, 2, 3, 8, 2, 0, None, 0, None) == seq_cabi.ERR_WORKSPACE

    def call(**change):
        c = seq_cabi.DeltaCall(T=70, B=2, Hk=2, Hv=4, Dk=16, Dv=8, scale=1.0, dtype=F32)
        for n in ("q", "k", "v", "g", "beta"):
            setattr(c, n, p)
        for n, value in change.items():
            setattr(c, n, value)
        return c

    delta = lambda ws=p, n=1 << 40, **change: lib.snnseq_gated_delta_fp(call(**change), p, p, ws, n, 1, None)
    assert delta(dtype=F64) == seq_cabi.ERR_UNSUPPORTED and delta(dtype=5) == seq_cabi.ERR_DTYPE
    for bad in ({"T": -1}, {"B": -1}, {"Hk": 0}, {"Hv": 3}, {"Dk": 129}, {"Dk": 0}, {"Dv": 0}, {"Dv": 65537},
                {"B": 65536}, {"Hv": 65536}, {"q": None}, {"beta": None}, {"T": seq_cabi.MAX_TOKENS + 1}):
        assert delta(**bad) == seq_cabi.ERR_ARG, bad
    assert delta(q=odd) == delta(state=odd) == seq_cabi.ERR_ALIGN
    assert delta(n=0) == delta(ws=None) == seq_cabi.ERR_WORKSPACE
    assert delta(B=0, q=None) == seq_cabi.OK
    assert lib.snnseq_gated_delta_fp(None, p, p, p, 0, 1, None) == seq_cabi.ERR_ARG
    saved, scratch = (lib.snnseq_gated_delta_saved_bytes(call(), b) for b in (1, 0))
    assert 0 < scratch < saved and lib.snnseq_gated_delta_saved_bytes(call(Dk=0), 1) == 0
    assert lib.snnseq_gated_delta_bp_workspace_bytes(call()) > 0
    strides = (ctypes.c_int64 * 3)(64, 32, 8)
    back = lambda s=strides, n=saved: lib.snnseq_gated_delta_bp(call(), p, n, p, s, p, p, p, p, p, p, p, p, 0, None)
    assert back(s=None) == seq_cabi.ERR_ARG and back() == seq_cabi.ERR_WORKSPACE
    step = lambda **change: lib.snnseq_gated_delta_step(call(**{"T": 1, "state": p, **change}), p, p, None)
    assert step(T=2) == step(state=None) == step(lengths=p) == step(v=None) == seq_cabi.ERR_ARG
    assert step(B=0) == seq_cabi.OK


def test_launches_hold_what_is_accepted():
    """Sizes whose launch would have more workgroups or threads than one can: refused, or worked on in another layout."""
    lib = seq_cabi.load()
    call = seq_cabi.DeltaCall(T=70, B=1024, Hk=4, Hv=4, Dk=1, Dv=65536, scale=1.0, dtype=F32)
    for n in ("q", "k", "v", "g", "beta"):
        setattr(call, n, 4096)
    assert lib.snnseq_gated_delta_saved_bytes(call, 1) == lib.snnseq_gated_delta_bp_workspace_bytes(call) == 0
    p = ctypes.c_void_p(4096)
    assert lib.snnseq_gated_delta_fp(call, p, p, p, 1 << 62, 1, None) == seq_cabi.ERR_ARG
    call.B = 512
    assert lib.snnseq_gated_delta_saved_bytes(call, 1) > 0
    # a sample of 4096 positions of one group of four is a workgroup's of 1024 threads, unless there are too many of them
    assert lib.snnseq_gn_act_workspace_bytes(F32, 1000, 4096, 4, 1, 0) == 0
    assert lib.snnseq_gn_act_workspace_bytes(F32, seq_cabi.MAX_TOKENS, 4096, 4, 1, 0) > 0


def test_helpers_reject_mismatched_buffers_before_any_launch():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    stat = torch.zeros(2, 2)
    with pytest.raises(ValueError, match="out has shape"):
        seq_cabi.embed_fp_into(torch.zeros(4, dtype=torch.long), torch.zeros(5, 6), torch.zeros(4, 5), 1.0)
    with pytest.raises(ValueError, match="workspace"):
        seq_cabi.embed_bp_into(torch.zeros(4, dtype=torch.long), torch.zeros(4, 6), torch.zeros(5, 6), 1.0, None)
    with pytest.raises(TypeError, match="token dtype"):
        seq_cabi.embed_fp_into(torch.zeros(4), torch.zeros(5, 6), torch.zeros(4, 6), 1.0)
    with pytest.raises(ValueError, match="mean has dtype"):
        seq_cabi.gn_act_fp_into(x, w, w, x.clone(), stat.double(), stat, 2, 1e-5, "silu")
    with pytest.raises(ValueError, match="grad_x has shape"):
        seq_cabi.gn_act_bp_into(x, w, w, stat, stat, x, x[:1], w, w, 2, "silu", None)
    q, g = torch.zeros(5, 2, 1, 4), torch.zeros(5, 2, 1)
    with pytest.raises(ValueError, match="beta has shape"):
        seq_cabi.delta_call(q, q, q, g, g[:4])
    with pytest.raises(ValueError, match="must be dense"):
        seq_cabi.delta_call(q.transpose(1, 3).contiguous().transpose(1, 3), q, q, g, g)
    with pytest.raises(ValueError, match="o has shape"):
        seq_cabi.gated_delta_fp_into(seq_cabi.delta_call(q, q, q, g, g), q[:4], None, None)
    with pytest.raises(ValueError, match="device tensor required"):
        seq_cabi.embed_fp_into(torch.zeros(4, dtype=torch.long), torch.zeros(5, 6), torch.zeros(4, 6), 1.0)


def test_python_surface():
    from snn_gpu_training_bptt_amd import snnlib_func as sf
    from snn_gpu_training_bptt_amd import snnlib_op as sop
    for name in ("embed", "embed_fp", "embed_bp", "gn_act", "gn_act_fp", "gn_act_bp", "gated_delta", "gated_delta_fp",
                 "gated_delta_bp", "gated_delta_step"):
        assert callable(getattr(sf.snnlib, name))
    assert sf.snnlib.__seq_abi_version__ == seq_cabi.ABI_VERSION
    for name in ("Embed", "GnAct", "GatedDelta"):
        assert issubclass(getattr(sop, name), torch.nn.Module)
    for name in ("embed_func", "gn_act_func", "gated_delta_func", "gated_delta_step"):
        assert callable(getattr(sf, name))
    embed, norm, delta = sop.Embed(11, 6, 2.0), sop.GnAct(2, 8), sop.GatedDelta()
    assert {n: tuple(t.shape) for n, t in embed.named_parameters()} == {"weight_embed": (11, 6)}
    assert {n: tuple(t.shape) for n, t in norm.named_parameters()} == {"weight_gn": (8,), "bias_gn": (8,)}
    assert delta.state_dict() == {}
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        embed(torch.zeros(3, 2, dtype=torch.long))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        norm(torch.zeros(3, 2, 8))


@pytest.mark.gpu
def test_through_the_c_abi_alone():
    """Same bits as the module's operators, from buffers the caller owns: outputs that held NaN, a workspace larger than
    asked for, and untouched memory behind every output."""
    from snn_gpu_training_bptt_amd import snnlib_func as sf
    lib = seq_cabi.load()
    gen = torch.Generator().manual_seed(0)
    nan = lambda *s, **k: torch.full(s, float("nan"), device="cuda", **k)
    tokens = torch.randint(-1, 9, (70,), generator=gen).cuda()
    weight, grad = torch.randn(9, 10, generator=gen).cuda(), torch.randn(70, 10, generator=gen).cuda()
    out, gw = nan(71, 10), nan(10, 10)
    seq_cabi.embed_fp_into(tokens, weight, out[:70], 0.5)
    seq_cabi.embed_bp_into(tokens, grad, gw[:9], 0.5, torch.full((5000,), 255, dtype=torch.uint8, device="cuda"))
    assert torch.equal(out[:70], sf.snnlib.embed_fp(tokens, weight, 0.5)) and bool(out[70].isnan().all())
    assert torch.equal(gw[:9], sf.snnlib.embed_bp(tokens, grad, 9, 0.5)) and bool(gw[9].isnan().all())

    x = torch.randn(6, 5, 12, generator=gen).cuda()
    w, b, gy = (torch.randn(*s, generator=gen).cuda() for s in ((12,), (12,), (6, 5, 12)))
    y, mean, rstd, gx, gwb = nan(7, 5, 12), nan(7, 3), nan(7, 3), nan(7, 5, 12), nan(3, 12)
    seq_cabi.gn_act_fp_into(x, w, b, y[:6], mean[:6], rstd[:6], 3, 1e-5, "gelu")
    need = lib.snnseq_gn_act_workspace_bytes(F32, 6, 5, 12, 3, 1)
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    seq_cabi.gn_act_bp_into(x, w, b, mean[:6], rstd[:6], gy, gx[:6], gwb[0], gwb[1], 3, "gelu", ws)
    as_layer = x.reshape(2, 3, 5, 12)
    m0, r0, y0 = sf.snnlib.gn_act_fp(as_layer, w, b, 3, 1e-5, "gelu")
    gx0, gw0, gb0 = sf.snnlib.gn_act_bp(as_layer, w, b, m0, r0, 3, "gelu", gy.reshape(2, 3, 5, 12))
    assert torch.equal(y[:6].reshape(y0.shape), y0) and torch.equal(gx[:6].reshape(gx0.shape), gx0)
    assert torch.equal(gwb[0], gw0) and torch.equal(gwb[1], gb0)
    assert bool(y[6].isnan().all()) and bool(gx[6].isnan().all()) and bool(mean[6].isnan().all()) and bool(gwb[2].isnan().all())
    assert bool((ws[need:] == 255).all())

    T, B, H, D = 70, 2, 2, 40
    q, k, v = (torch.nn.functional.normalize(torch.randn(T, B, H, D, generator=gen), dim=-1).cuda() for _ in range(3))
    g, beta = -torch.rand(T, B, H, generator=gen).cuda(), torch.rand(T, B, H, generator=gen).cuda()
    call = seq_cabi.delta_call(q, k, v, g, beta, scale=0.3)
    o, last = nan(T + 1, B, H, D), nan(B + 1, H, D, D)
    for for_backward in (True, False):
        need = lib.snnseq_gated_delta_saved_bytes(call, int(for_backward))
        saved = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
        seq_cabi.gated_delta_fp_into(call, o[:T], last[:B], saved, for_backward)
        o0, last0, _ = sf.snnlib.gated_delta_fp(q, k, v, g, beta, None, None, 0.3)
        assert torch.equal(o[:T], o0) and torch.equal(last[:B], last0)
        assert bool(o[T].isnan().all()) and bool(last[B].isnan().all()) and bool((saved[need:] == 255).all())
