"""ctypes view of the token-layer C ABI in ``include/snnlib_seq.h`` (``libsnnlif_gfx950.so``).

The counterpart of ``lif_cabi`` for embedding, group norm with an activation and the gated delta rule: raw
device pointers, sizes and a stream handle.  The helpers at the bottom unwrap ``torch.Tensor`` arguments and check what
the C side cannot see -- that every buffer is as large as the sizes handed over say.
"""
import ctypes

from . import lif_cabi
from .lif_cabi import (DTYPE_BF16, DTYPE_F32, DTYPE_F64, ERR_ALIGN, ERR_ARG, ERR_DTYPE, ERR_UNSUPPORTED,  # noqa: F401
                       ERR_WORKSPACE, OK, SnnlifError)

ABI_VERSION = 1
TOKEN_I32, TOKEN_I64 = 0, 1
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
MAX_TOKENS, MAX_CHANNELS, MAX_KEY, MAX_VALUE, MAX_HEADS = 8388608, 1048576, 128, 65536, 65535

_vp, _i64, _int, _sz, _f64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t, ctypes.c_double


class DeltaCall(ctypes.Structure):
    """``snnseq_delta``."""
    _fields_ = ([(n, _i64) for n in ("T", "B", "Hk", "Hv", "Dk", "Dv")]
                + [(n, _i64 * 3) for n in ("q_strides", "k_strides", "v_strides")]
                + [("scale", _f64)] + [(n, _vp) for n in ("q", "k", "v", "g", "beta", "state", "lengths")]
                + [("dtype", _int)])


_call = ctypes.POINTER(DeltaCall)
# name -> (restype, argtypes); must list every symbol include/snnlib_seq.h declares.
SYMBOLS = {
    "snnseq_abi_version": (_int, []),
    "snnseq_embed_fp": (_int, [_vp] * 3 + [_int, _int, _i64, _i64, _i64, _i64, _f64, _vp]),
    "snnseq_embed_bp_workspace_bytes": (_sz, [_int, _i64, _i64, _i64]),
    "snnseq_embed_bp": (_int, [_vp] * 3 + [_int, _int, _i64, _i64, _i64, _f64, _vp, _sz, _vp]),
    "snnseq_gn_act_workspace_bytes": (_sz, [_int, _i64, _i64, _i64, _i64, _int]),
    "snnseq_gn_act_fp": (_int, [_vp] * 6 + [_int, _i64, _i64, _i64, _i64, _f64, _int, _vp, _sz, _vp]),
    "snnseq_gn_act_bp": (_int, [_vp] * 9 + [_int, _i64, _i64, _i64, _i64, _int, _vp, _sz, _vp]),
    "snnseq_gated_delta_saved_bytes": (_sz, [_call, _int]),
    "snnseq_gated_delta_fp": (_int, [_call, _vp, _vp, _vp, _sz, _int, _vp]),
    "snnseq_gated_delta_bp_workspace_bytes": (_sz, [_call]),
    "snnseq_gated_delta_bp": (_int, [_call, _vp, _sz, _vp, ctypes.POINTER(_i64)] + [_vp] * 8 + [_sz, _vp]),
    "snnseq_gated_delta_step": (_int, [_call, _vp, _vp, _vp]),
}

_typed = False


def load():
    """The library of ``lif_cabi``, with the token-layer entry points typed."""
    global _typed
    lib = lif_cabi.load()
    if not _typed:
        for name, (restype, argtypes) in SYMBOLS.items():
            fn = getattr(lib, name)
            fn.restype = restype
            fn.argtypes = argtypes
        _typed = True
    return lib


# ---- thin tensor-unwrapping helpers (used by tests; torch is plumbing only) ----------------------------------

def _require(name, t, shape, dtype):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")


def _require_workspace(workspace, need, where):
    import torch
    if need and (workspace is None or workspace.dtype != torch.uint8 or workspace.numel() < need):
        raise ValueError(f"{where} needs a uint8 workspace of {need} bytes")


def _pointer(t):
    return ctypes.c_void_p(None if t is None else t.data_ptr())


def _token_dtype(tokens):
    import torch
    codes = {torch.int32: TOKEN_I32, torch.int64: TOKEN_I64}
    if tokens.dtype not in codes:
        raise TypeError(f"unsupported token dtype {tokens.dtype}")
    return codes[tokens.dtype]


def embed_fp_into(tokens, weight, out, scale):
    """``out`` [N, C] from dense ``tokens`` [N] and ``weight`` [V, C]."""
    lib, token_dtype = load(), _token_dtype(tokens)
    _require("out", out, (tokens.numel(), weight.shape[1]), weight.dtype)
    lif_cabi._require_dense_gpu(tokens, weight, out)
    lif_cabi._check(lib.snnseq_embed_fp(_pointer(tokens), _pointer(weight), _pointer(out),
                                        lif_cabi._torch_dtype_code(weight), token_dtype, tokens.numel(),
                                        weight.shape[0], weight.shape[1], weight.shape[1], float(scale),
                                        lif_cabi._stream_handle(weight)), "snnseq_embed_fp")


def embed_bp_into(tokens, grad, grad_weight, scale, workspace):
    lib, token_dtype = load(), _token_dtype(tokens)
    _require("grad", grad, (tokens.numel(), grad_weight.shape[1]), grad_weight.dtype)
    code = lif_cabi._torch_dtype_code(grad)
    need = lib.snnseq_embed_bp_workspace_bytes(code, tokens.numel(), *grad_weight.shape)
    _require_workspace(workspace, need, "snnseq_embed_bp")
    lif_cabi._require_dense_gpu(tokens, grad, grad_weight, workspace)
    lif_cabi._check(lib.snnseq_embed_bp(_pointer(tokens), _pointer(grad), _pointer(grad_weight), code,
                                        token_dtype, tokens.numel(), *grad_weight.shape, float(scale),
                                        _pointer(workspace), workspace.numel(), lif_cabi._stream_handle(grad)),
                    "snnseq_embed_bp")


def _statistics_dtype(x):
    import torch
    return torch.float64 if x.dtype == torch.float64 else torch.float32


def gn_act_fp_into(x, weight, bias, y, mean, rstd, groups, eps, act, workspace=None):
    """``x``, ``y`` dense [S, P, C]; ``mean``, ``rstd`` [S, groups]."""
    lib = load()
    S, P, C = x.shape
    for name, t in (("weight", weight), ("bias", bias)):
        _require(name, t, (C,), x.dtype)
    _require("y", y, x.shape, x.dtype)
    for name, t in (("mean", mean), ("rstd", rstd)):
        _require(name, t, (S, groups), _statistics_dtype(x))
    code = lif_cabi._torch_dtype_code(x)
    _require_workspace(workspace, lib.snnseq_gn_act_workspace_bytes(code, S, P, C, groups, 0), "snnseq_gn_act_fp")
    lif_cabi._require_dense_gpu(x, weight, bias, y, mean, rstd, workspace)
    lif_cabi._check(lib.snnseq_gn_act_fp(*(_pointer(t) for t in (x, weight, bias, y, mean, rstd)), code, S, P, C, groups,
                                         float(eps), ACTS[act], _pointer(workspace),
                                         0 if workspace is None else workspace.numel(), lif_cabi._stream_handle(x)),
                    "snnseq_gn_act_fp")


def gn_act_bp_into(x, weight, bias, mean, rstd, grad_y, grad_x, grad_weight, grad_bias, groups, act, workspace):
    lib = load()
    S, P, C = x.shape
    for name, t in (("weight", weight), ("bias", bias), ("grad_weight", grad_weight), ("grad_bias", grad_bias)):
        _require(name, t, (C,), x.dtype)
    for name, t in (("grad_y", grad_y), ("grad_x", grad_x)):
        _require(name, t, x.shape, x.dtype)
    for name, t in (("mean", mean), ("rstd", rstd)):
        _require(name, t, (S, groups), _statistics_dtype(x))
    code = lif_cabi._torch_dtype_code(x)
    _require_workspace(workspace, lib.snnseq_gn_act_workspace_bytes(code, S, P, C, groups, 1), "snnseq_gn_act_bp")
    tensors = (x, weight, bias, mean, rstd, grad_y, grad_x, grad_weight, grad_bias)
    lif_cabi._require_dense_gpu(*tensors, workspace)
    lif_cabi._check(lib.snnseq_gn_act_bp(*(_pointer(t) for t in tensors), code, S, P, C, groups, ACTS[act],
                                         _pointer(workspace), workspace.numel(), lif_cabi._stream_handle(x)),
                    "snnseq_gn_act_bp")


def delta_call(q, k, v, g, beta, state=None, lengths=None, scale=1.0):
    """The ``snnseq_delta`` of ``[T, B, H, D]`` operands whose rows are dense; keep the tensors alive while it is used."""
    import torch
    T, B, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    _require("k", k, q.shape, q.dtype)
    _require("v", v, (T, B, Hv, Dv), q.dtype)
    for name, t in (("g", g), ("beta", beta)):
        _require(name, t, (T, B, Hv), torch.float32)
    if state is not None:
        _require("state", state, (B, Hv, Dk, Dv), torch.float32)
    if lengths is not None:
        _require("lengths", lengths, (B,), torch.int32)
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"the rows of {name} must be dense")
    for t in (g, beta, state, lengths):
        if t is not None and not t.is_contiguous():
            raise ValueError("dense (contiguous) tensor required")
    strides = lambda t: (_i64 * 3)(*t.stride()[:3])
    return DeltaCall(T=T, B=B, Hk=Hk, Hv=Hv, Dk=Dk, Dv=Dv, q_strides=strides(q), k_strides=strides(k),
                     v_strides=strides(v), scale=float(scale), q=_pointer(q), k=_pointer(k), v=_pointer(v), g=_pointer(g),
                     beta=_pointer(beta), state=_pointer(state), lengths=_pointer(lengths),
                     dtype=lif_cabi._torch_dtype_code(q))


def gated_delta_fp_into(call, o, state_out, saved, for_backward=True):
    """``o`` dense [T, B, Hv, Dv] of the operands' type, ``state_out`` fp32 [B, Hv, Dk, Dv] or None."""
    import torch
    lib = load()
    if tuple(o.shape) != (call.T, call.B, call.Hv, call.Dv) or lif_cabi._torch_dtype_code(o) != call.dtype:
        raise ValueError(f"o has shape {tuple(o.shape)} and dtype {o.dtype}, which are not those of the call")
    if state_out is not None:
        _require("state_out", state_out, (call.B, call.Hv, call.Dk, call.Dv), torch.float32)
    _require_workspace(saved, lib.snnseq_gated_delta_saved_bytes(call, int(for_backward)), "snnseq_gated_delta_fp")
    lif_cabi._require_dense_gpu(o, state_out, saved)
    lif_cabi._check(lib.snnseq_gated_delta_fp(call, _pointer(o), _pointer(state_out), _pointer(saved),
                                              0 if saved is None else saved.numel(), int(for_backward),
                                              lif_cabi._stream_handle(o)), "snnseq_gated_delta_fp")
