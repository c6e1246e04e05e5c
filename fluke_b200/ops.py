"""Tensor-level operator interface: one function per C entry point, same name without the
`fluke_` prefix, same argument meaning and the same error behaviour (void functions exit the
process on a bad dimension, int functions raise on a non-zero return). Inputs must be
contiguous CUDA tensors; nothing here computes on the host, and no call records anything for
autograd. The work of a call (checks, output
allocation, the C call) is done by the extension module (csrc/native_ops.cpp); what is not called
per step goes through ctypes.
"""
import contextlib
import ctypes

import torch

from . import lib as _lib

TX_DIMS = dict(d_model=512, dim_feedforward=2048, nhead=8, head_dim=64)


def _L():
    return _lib.load()


class _Native:
    """The extension module, loaded (and built if it is missing) at the first call of an operator."""

    def __getattr__(self, name):
        fn = getattr(_lib.native(), name)
        setattr(self, name, fn)
        return fn


_N = _Native()


def _dev(*ts):
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("fluke_b200.ops needs CUDA tensors (there is no CPU fallback)")
        if not t.is_contiguous():
            raise RuntimeError("fluke_b200.ops needs contiguous tensors")


def _p(t):
    return 0 if t is None else t.data_ptr()


def _check(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} failed: rc={rc} {_L().fluke_last_error().decode()}")


def set_stream(stream=None):
    """Route later launches of this thread to `stream` (torch.cuda.Stream) or back to the legacy default stream."""
    _L().fluke_set_stream(0 if stream is None else stream.cuda_stream)


@contextlib.contextmanager
def on_stream(stream):
    """Routes this thread's launches to `stream` inside a `with` block, and puts back what was set. The setting is of a thread, and torch runs
    backward functions on threads of its own: they call under `with on_stream(torch.cuda.current_stream(device))`."""
    before = _L().fluke_get_stream()
    set_stream(stream)
    try:
        yield
    finally:
        _L().fluke_set_stream(before)


# ---- memory-bound kernels -----------------------------------------------------------------

def rmsnorm(x, residual, weight, alpha, eps, out=None):
    return _N.rmsnorm(x, residual, weight, alpha, eps, out)


def rmsnorm_quant_int8(x, weight, residual_i8, residual_scale, alpha, eps):
    """In place on (residual_i8, residual_scale)."""
    return _N.rmsnorm_quant(x, weight, residual_i8, residual_scale, alpha, eps, False)


def rmsnorm_quant_fp8(x, weight, residual_u8, residual_scale, alpha, eps):
    return _N.rmsnorm_quant(x, weight, residual_u8, residual_scale, alpha, eps, True)


def quant_int8(x, out=None, scale=None):
    return _N.quant(x, out, scale, False)


def quant_fp8(x, out=None, scale=None):
    return _N.quant(x, out, scale, True)


def dequant_transpose(x, scale, fp8=False):
    """[T,N,C] int8 / e4m3 bytes -> f16 [N,T,C]."""
    return _N.dequant_transpose(x, scale, fp8)


def rotary_emb_(x_ptr, sin, cos, batch, seq_len, n_heads, head_dim, width, sb, ss, sh):
    """In place on the f16 tensor starting at device address x_ptr (strides in elements)."""
    _N.rotary_emb(x_ptr, sin, cos, batch, seq_len, n_heads, head_dim, width, sb, ss, sh)


def rotary_qkv_(qkv, sin, cos, width):
    """Rotate the q and k chunks of qkv [N, seq, 3, heads, head_dim] in place, passing the full
    qkv strides (the call pattern of test/test_rotary_gpu.py:26-38)."""
    return _N.rotary_qkv(qkv, sin, cos, width)


def silu_mul(x):
    return _N.silu_mul(x)


def flstm_step(scratch, ih_t, cell, hh_next=None):
    return _N.flstm_step(scratch, ih_t, cell, hh_next)


# ---- fused transformer kernels ------------------------------------------------------------

def int8_select(device_index=0, max_seq=2048, **dims):
    d = dict(TX_DIMS, **dims)
    b = _L().fluke_int8_select(device_index, _lib.fluke_dims_t(d["d_model"], d["dim_feedforward"],
                                                               d["nhead"], d["head_dim"], max_seq))
    return b  # None when unsupported (the caller keeps fp16, as with the reference)


def fp8_select(device_index=0, max_seq=2048, **dims):
    d = dict(TX_DIMS, **dims)
    return _L().fluke_fp8_select(device_index, _lib.fluke_dims_t(d["d_model"], d["dim_feedforward"],
                                                                d["nhead"], d["head_dim"], max_seq))


def qkv_rotary_i8(backend, a_i8, wqkv_i8, scale_a, scale_b, sin, cos, seqlen, out=None):
    return _N.qkv_rotary(backend, a_i8, wqkv_i8, scale_a, scale_b, sin, cos, seqlen, out, 0, wqkv_i8.size(0))


def gated_mlp_i8(backend, a_i8, gate_i8, up_i8, scale_a, scale_gate, scale_up, out=None):
    return _N.gated_mlp(backend, a_i8, gate_i8, up_i8, scale_a, scale_gate, scale_up, out, 0, gate_i8.size(0))


def qkv_rotary_fp8(backend, a_fp8, w_fp8, scale_a, scale_b, sin, cos, seqlen, plain=False, out=None):
    """w_fp8: PRESHUFFLED bytes (plain=False, the reference ABI) or row-major [N,K] (plain=True)."""
    return _N.qkv_rotary(backend, a_fp8, w_fp8, scale_a, scale_b, sin, cos, seqlen, out, 2 if plain else 1,
                         3 * TX_DIMS["d_model"])


def gated_mlp_fp8(backend, a_fp8, gate_fp8, up_fp8, scale_a, scale_gate, scale_up, plain=False, out=None):
    return _N.gated_mlp(backend, a_fp8, gate_fp8, up_fp8, scale_a, scale_gate, scale_up, out, 2 if plain else 1,
                        TX_DIMS["dim_feedforward"])


# ---- base GEMMs (additive) ----------------------------------------------------------------

def gemm_i8(a_i8, b_i8, scale_a, scale_b, const_scale_a=0.0):
    return _N.gemm_i8(a_i8, b_i8, scale_a, scale_b, const_scale_a)


def gemm_i8_s32(a_i8, b_i8):
    _dev(a_i8, b_i8)
    m, k = a_i8.shape
    n = b_i8.size(0)
    out = torch.empty(m, n, dtype=torch.int32, device=a_i8.device)
    _check(_L().fluke_gemm_i8_s32_gpu(_p(out), _p(a_i8), _p(b_i8), m, n, k), "fluke_gemm_i8_s32_gpu")
    return out


def gemm_fp8(a_fp8, b_fp8_nk, scale_a, scale_b):
    return _N.gemm_fp8(a_fp8, b_fp8_nk, scale_a, scale_b)


def fp8_unshuffle(w_preshuffled, n, k):
    _dev(w_preshuffled)
    out = torch.empty(n, k, dtype=torch.uint8, device=w_preshuffled.device)
    _check(_L().fluke_fp8_unshuffle_gpu(_p(out), _p(w_preshuffled), n, k), "fluke_fp8_unshuffle_gpu")
    return out


# ---- microscaled 4-bit floating point (additive) --------------------------------------------
# A quantised matrix is (codes, scale) in mxfp4 and (codes, scale, row_scale) in nvfp4: uint8 codes
# [rows, cols / 2], uint8 block scales [ceil(rows / 128), ceil(blocks / 4), 512] in the tiles that fluke.h
# describes, f32 row scales [rows]. Activations are f16 or bf16. A wrong type, shape, device or
# alignment raises; the calls run on the tensors' device.

def quant_mxfp4(x):
    """x [rows, cols] -> (codes, scale): blocks of 32 under a power of two."""
    return _N.quant_fp4(x, False)


def quant_nvfp4(x):
    """x [rows, cols] -> (codes, scale, row_scale): blocks of 16 under an e4m3 scale, rows under a power of two."""
    return _N.quant_fp4(x, True)


def dequant_mxfp4(codes, scale, dtype=torch.float16):
    return _N.dequant_fp4(codes, scale, None, dtype, False)


def dequant_nvfp4(codes, scale, row_scale, dtype=torch.float16):
    return _N.dequant_fp4(codes, scale, row_scale, dtype, True)


def gemm_mxfp4(a, a_scale, b, b_scale, dtype=torch.float16):
    """[M, N] = a [M, K] @ b [N, K]^T of two quantised matrices."""
    return _N.gemm_fp4(a, a_scale, None, b, b_scale, None, None, None, None, dtype, False, False)


def gemm_nvfp4(a, a_scale, a_row, b, b_scale, b_row, dtype=torch.float16):
    return _N.gemm_fp4(a, a_scale, a_row, b, b_scale, b_row, None, None, None, dtype, True, False)


def gated_mlp_mxfp4(a, a_scale, gate, gate_scale, up, up_scale, dtype=torch.float16):
    """[M, N] = silu(a @ gate^T) * (a @ up^T), gate and up [N, K]."""
    return _N.gemm_fp4(a, a_scale, None, gate, gate_scale, None, up, up_scale, None, dtype, False, True)


def gated_mlp_nvfp4(a, a_scale, a_row, gate, gate_scale, gate_row, up, up_scale, up_row, dtype=torch.float16):
    return _N.gemm_fp4(a, a_scale, a_row, gate, gate_scale, gate_row, up, up_scale, up_row, dtype, True, True)


def rmsnorm_block(x, residual, post_weight, gate, pre_weight, alpha, eps, seqlen=0, quant=None, residual_out=None):
    """Norms around a block: stream = alpha * residual + gate * norm(x, post_weight), then norm(stream, pre_weight)
    for the next block, as 16-bit values (quant None) or quantised: "mxfp4", "nvfp4", or "int8" (int8 codes) and "e4m3"
    (fp8 bytes) under an f32 scale per row, as the 8-bit products take them (up to 1024 columns; wider rows have no product here). gate [cols], or
    [ceil(rows / seqlen), cols] with seqlen > 0. post_weight, gate and pre_weight may be None. Returns the
    stream (written to `residual_out`, which may be `residual` or `x`, or to a new tensor) followed by the
    next block's input: (stream, out), (stream, codes, scale[, row_scale]) with the row scales alone for 8 bits, or (stream,) without
    pre_weight."""
    if quant not in _QUANT:
        raise ValueError(f"quant is None, 'mxfp4', 'nvfp4', 'int8' or 'e4m3', not {quant!r}")
    return _N.rmsnorm_block(x, residual, post_weight, gate, pre_weight, alpha, eps, seqlen, _QUANT[quant], residual_out)


_QUANT = {None: 0, "mxfp4": _lib.FP4_MX, "nvfp4": _lib.FP4_NV, "int8": _lib.ROW_INT8, "e4m3": _lib.ROW_FP8}


# ---- 16-bit product with an epilogue, gated linear recurrence (additive) ----------------------
# f16 or bf16; inputs may be views whose last dimension is dense (columns of a wider tensor, transposed leading
# dimensions). A wrong type, shape, device, stride or alignment raises; the calls run on the tensors' device.

def linear(x, weight, bias=None, activation=None, residual=None, alpha=1.0, out=None):
    """[M, N] = activation(x [M, K] @ weight [N, K]^T + bias [N]) + alpha * residual [M, N], rounded once. activation: None,
    "relu", "silu", "gelu", "tanh" or "sigmoid". K and N are multiples of 8, rows begin on 16 bytes. `out` may be
    `residual`, else it lies apart from the inputs."""
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"activation is None, 'relu', 'silu', 'gelu', 'tanh' or 'sigmoid', not {activation!r}")
    return _N.linear(x, weight, bias, _lib.ACTIVATIONS[activation], residual, alpha, out)


def linear_recurrence(gate, value, h0=None, lengths=None, reverse=False, save=False, out=None, h_last=None):
    """h_t = f_t h_{t-1} + (1 - f_t) value_t with f = sigmoid(gate), per chunk and channel of gate and value [T, B, H], over t = 0 ..
    T-1, or T-1 .. 0 with `reverse`. h0 f32 [B, H] (None: zeros). With lengths (int32 [B]) the steps t >= lengths[b] are not
    taken and their output is zero. Returns (out, h_last), out as `value` in type and, where it is new, in the order of
    its leading dimensions, h_last f32 [B, H] (may be given, as h0 itself too); with `save` also the states that
    linear_recurrence_backward needs."""
    return _N.linear_recurrence(gate, value, h0, lengths, reverse, save, out, h_last)


def linear_recurrence_backward(grad, gate, value, states, grad_last=None, lengths=None, reverse=False):
    """Gradients (of gate, of value, of h0) from those of out (grad [T, B, H]) and of h_last (f32 [B, H] or None: zeros), with
    the inputs of the forward call and the states it saved."""
    return _N.linear_recurrence_backward(grad, gate, value, states, grad_last, lengths, reverse)


# ---- factored LSTM (additive) ---------------------------------------------------------------

def down_proj_i8(a_i8, w_i8, scale_a, scale_b, out=None):
    """f16 [M,N] = int8 GEMM * (sa*sb); scale_a None = the fixed 1/127 of an int8 hidden state."""
    return _N.down_proj(a_i8, w_i8, scale_a, scale_b, out, False)


def down_proj_fp8(a_fp8, w_fp8_nk, scale_a, scale_b, out=None):
    """f16 [M,N] = (e4m3 GEMM * sa[m]) * sb[n]; a_fp8 [M,K], w_fp8_nk [N,K] as uint8 e4m3 bytes."""
    return _N.down_proj(a_fp8, w_fp8_nk, scale_a, scale_b, out, True)


def factored_lstm_step_i8(A, W4, bias4, c, h_out=None, fp8_export_name=False):
    """A f16 [B,Kc]; W4 f16 [4H,Kc] (gate-major i,f,g,o); bias4 f32 [4H]; c f32 [B,H] in place."""
    return _N.lstm_step(A, W4, bias4, c, h_out, fp8_export_name)


def factored_lstm_layer_i8(x_i8, x_scale, dn_ih, dn_ih_scale, dn_hh, dn_hh_scale, w_up, bias, c, h,
                           reverse=False, h_out=None, workspace=None, phase_mask=7):
    """One layer over x_i8 [T,B,H]; c (f32 [B,H]) and h (int8 [B,H]) are state, updated in place.
    phase_mask != 7 launches only some kernel classes (timing aid, see fluke.h)."""
    _dev(x_i8, x_scale, dn_ih, dn_ih_scale, dn_hh, dn_hh_scale, w_up, bias, c, h)
    t, b, hd = x_i8.shape
    r = dn_ih.size(0)
    need = _L().fluke_factored_lstm_layer_workspace(t, b, hd, r)
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=x_i8.device)
    h_out = torch.empty(t, b, hd, dtype=torch.int8, device=x_i8.device) if h_out is None else h_out
    layer = _lib.fluke_flstm_layer_t(t, b, hd, r, 1 if reverse else 0, _p(x_i8), _p(x_scale),
                                     _p(dn_ih), _p(dn_ih_scale), _p(dn_hh), _p(dn_hh_scale),
                                     _p(w_up), _p(bias), _p(c), _p(h), _p(h_out),
                                     _p(workspace), workspace.numel())
    if phase_mask == 7:
        _check(_L().fluke_factored_lstm_layer_i8_gpu(ctypes.byref(layer)), "fluke_factored_lstm_layer_i8_gpu")
    else:
        _check(_L().fluke_factored_lstm_layer_phases_gpu(ctypes.byref(layer), phase_mask),
               "fluke_factored_lstm_layer_phases_gpu")
    return h_out
