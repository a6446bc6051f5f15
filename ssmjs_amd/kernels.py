"""Kernel-level entry points of libssm_hip.so on torch device tensors.

torch supplies device memory and the current HIP stream only; every computation runs in
the HIP kernels of libssm_hip.so. All tensors must live on a HIP device; a CPU tensor is an
error (there is no CPU path).

Shapes (row-major):
  causal_conv1d    x (B,L,C) [row stride may exceed C], w (C,K) -> y (B,L,C)
  selective_scan   u, dt, z (B,L,D); B, C (B,L,N); A (D,N); state (B,D,N)
  ssd_chunk_scan   x (B,L,H,P); dt (B,L,H); B, C (B,L,G,N); A (H); state (B,H,P,N)
  linear_attention q (B,L,H,K); k (B,L,G,K); v (B,L,G,V); g (H); state (B,H,V,K)
  linear_i8/q8     x (M,K), W (N,K) -> y (M,N)
"""
from __future__ import annotations

import torch

from . import _lib
from .backend import sample_supported  # noqa: F401  (re-export)

_NULL = None
_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _p(t):
    """Device pointer of a tensor (None -> NULL)."""
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("ssmjs_amd kernels need HIP device tensors (no CPU path)")
    return t.data_ptr()


def _stream():
    """Handle of the current device's current stream, without a Stream object around it (1 us of
    each call) where torch has the calls for that."""
    if _device is None or _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(_device())


def _scratch(nbytes, device):
    """A call's workspace as (tensor or None, bytes): shapes that need none pay no allocation."""
    if nbytes == 0:
        return None, 0
    return torch.empty(nbytes, device=device, dtype=torch.uint8), nbytes


def _rows(t, width):
    """Row stride (elements between consecutive time steps) of a (..., width) view whose
    last dim is contiguous and whose leading dims flatten to rows."""
    if t.stride(-1) != 1:
        raise ValueError("last dimension must be contiguous")
    return t.stride(-2) if t.dim() >= 2 else width


def _seq_ld(t):
    """Row stride of a (B,L,X) view whose sequences follow one another."""
    s = t.stride()
    if len(s) == 3 and s[0] != t.shape[1] * s[1] and t.shape[1] > 1:
        raise ValueError("row-strided (B,L,X) views only")
    return s[1]


def _f32(t):
    if t is not None and t.dtype != torch.float32:
        raise TypeError(f"expected float32, got {t.dtype}")
    return t


def causal_conv1d(x, w, bias=None, silu=True, state_in=None, state_out=None, out=None):
    B, L, Cc = x.shape
    K = w.shape[1]
    _f32(x)
    y = out if out is not None else torch.empty(B, L, Cc, device=x.device, dtype=torch.float32)
    sb, ldx, sc = x.stride()
    if sc != 1 or (L > 1 and sb != L * ldx):
        raise ValueError("x must be a row-strided (B,L,C) view")
    _lib.call("ssm_causal_conv1d", _p(x), ldx, _p(w.contiguous()), _p(bias), _p(y), y.stride(1),
              B, L, Cc, K, int(silu), _p(state_in), _p(state_out), _stream())
    return y


def conv1d_update(x, w, bias, state, silu=True, out=None):
    B, Cc = x.shape
    y = out if out is not None else torch.empty(B, Cc, device=x.device, dtype=torch.float32)
    _lib.call("ssm_conv1d_update", _p(x), x.stride(0), _p(w.contiguous()), _p(bias), _p(y),
              y.stride(0), _p(state), B, Cc, w.shape[1], int(silu), _stream())
    return y


def selective_scan(u, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, softplus=True, h0=None,
                   hT=None, out=None):
    B, L, Dd = u.shape
    N = A.shape[1]
    y = out if out is not None else torch.empty(B, L, Dd, device=u.device, dtype=torch.float32)
    ws, nbytes = _scratch(_lib.lib().ssm_selective_scan_workspace(B, L, Dd, N), u.device)
    _lib.call("ssm_selective_scan", _p(u), _seq_ld(u), _p(dt), _seq_ld(dt), _p(dt_bias),
              int(softplus), _p(A.contiguous()), _p(Bm), _seq_ld(Bm), _p(Cm), _seq_ld(Cm),
              _p(D), _p(z), _seq_ld(z) if z is not None else 0, _p(y), y.stride(1), B, L, Dd, N,
              _p(h0), _p(hT), _p(ws), nbytes, _stream())
    return y


def m1_state_update(x, dt, A, Bm, Cm, D, z, dt_bias, h, softplus=True, out=None):
    B, Dd = x.shape
    N = A.shape[1]
    y = out if out is not None else torch.empty(B, Dd, device=x.device, dtype=torch.float32)
    _lib.call("ssm_m1_state_update", _p(x), x.stride(0), _p(dt), dt.stride(0), _p(dt_bias),
              int(softplus), _p(A.contiguous()), _p(Bm), Bm.stride(0), _p(Cm), Cm.stride(0),
              _p(D), _p(z), z.stride(0) if z is not None else 0, _p(y), y.stride(0), _p(h), B, Dd,
              N, _stream())
    return y


def ssd_workspace(B, L, H, P, G, N, device):
    n = _lib.lib().ssm_ssd_workspace(B, L, H, P, G, N)
    return torch.empty(max(n, 4), device=device, dtype=torch.uint8)


def ssd_chunk_scan(x, dt, A, Bm, Cm, D=None, dt_bias=None, softplus=True, dt_min=0.0,
                   dt_max=float("inf"), h0=None, hT=None, out=None, workspace=None):
    """x (B,L,H,P), Bm/Cm (B,L,G,N) in float32 or bfloat16 (same dtype); y is float32."""
    B, L, H, P = x.shape
    G, N = Bm.shape[2], Bm.shape[3]
    if x.dtype == torch.float32:
        dtype = _lib.SSM_F32
    elif x.dtype == torch.bfloat16:
        dtype = _lib.SSM_BF16
    else:
        raise TypeError("x must be float32 or bfloat16")
    if Bm.dtype != x.dtype or Cm.dtype != x.dtype:
        raise TypeError("x, B and C must share a dtype")
    y = out if out is not None else torch.empty(B, L, H, P, device=x.device, dtype=torch.float32)
    if workspace is not None:
        ws, nbytes = workspace, workspace.numel()
    else:
        ws, nbytes = _scratch(_lib.lib().ssm_ssd_workspace(B, L, H, P, G, N), x.device)
    ldx = x.stride(1)
    _lib.call("ssm_ssd_chunk_scan", dtype, _p(x), ldx, _p(dt), dt.stride(1), _p(dt_bias),
              int(softplus), float(dt_min), float(dt_max), _p(A), _p(Bm), Bm.stride(1), _p(Cm),
              Cm.stride(1), _p(D), _p(y), y.stride(1), B, L, H, P, G, N, _p(h0), _p(hT), _p(ws),
              nbytes, _stream())
    return y


def m2_state_update(x, dt, A, Bm, Cm, D, dt_bias, h, z=None, softplus=True, dt_min=0.0,
                    dt_max=float("inf"), out=None):
    """x (B,H,P); dt (B,H); Bm, Cm (B,G,N); h (B,H,P,N) updated in place."""
    B, H, P = x.shape
    G, N = Bm.shape[1], Bm.shape[2]
    y = out if out is not None else torch.empty(B, H, P, device=x.device, dtype=torch.float32)
    _lib.call("ssm_m2_state_update", _p(x), x.stride(0), _p(dt), dt.stride(0), _p(dt_bias),
              int(softplus), float(dt_min), float(dt_max), _p(A), _p(Bm), Bm.stride(0), _p(Cm),
              Cm.stride(0), _p(D), _p(z), z.stride(0) if z is not None else 0, _p(y), y.stride(0),
              _p(h), B, H, P, G, N, _stream())
    return y


def rmsnorm(x, w, eps=1e-5, out=None):
    M, n = x.shape
    y = out if out is not None else torch.empty_like(x)
    _lib.call("ssm_rmsnorm", _p(x), x.stride(0), _p(w), _p(y), y.stride(0), M, n, float(eps),
              _stream())
    return y


def argmax(x, out=None):
    """Row-wise greedy pick (ssm_argmax): lowest index among equal maxima, NaN never wins."""
    rows, n = x.shape
    o = out if out is not None else torch.empty(rows, dtype=torch.int32, device=x.device)
    _lib.call("ssm_argmax", _p(x), x.stride(0), rows, n, _p(o), _stream())
    return o


def sample_workspace(rows, n, device):
    """Workspace for sample (ssm_sample_workspace bytes)."""
    return torch.empty(max(1, _lib.lib().ssm_sample_workspace(rows, n)), dtype=torch.uint8,
                       device=device)


def sample(x, u, temperature=1.0, topK=50, topP=0.9, out=None, workspace=None):
    """sampleToken per row on the device (ssm_sample, src/session/streaming.ts:53-97).

    x: (rows, n) fp32 logits; u: (rows,) float64 draws in [0, 1) (Math.random()). Returns
    (rows,) int32 picks. Raises for n > 262144 or min(topK, n) > 1024."""
    rows, n = x.shape
    assert u.dtype == torch.float64 and u.numel() == rows and u.is_contiguous()
    o = out if out is not None else torch.empty(rows, dtype=torch.int32, device=x.device)
    ws = workspace if workspace is not None else sample_workspace(rows, n, x.device)
    _lib.call("ssm_sample", _p(x), x.stride(0), rows, n, float(temperature), int(topK),
              float(topP), _p(u), _p(o), _p(ws), ws.numel(), _stream())
    return o


def linear_rows_workspace(M, N, K, device):
    """Split-K workspace for linear_rows (None when the shape never splits)."""
    n = _lib.lib().ssm_linear_rows_workspace(M, N, K)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def linear_rows(x, W, mode=0, g=None, z=None, eps=1e-5, out=None, beta=0.0, workspace=None):
    """y = beta*y + s * p(x) W^T for M <= 64 rows (ssm_linear_rows): mode 0 plain, 1 RMSNorm
    (weight g), 2 gated RMSNorm (z, weight g). `workspace` (linear_rows_workspace) lets the
    kernel split K; without it the kernel runs unsplit."""
    M, K = x.shape
    N = W.shape[0]
    y = out if out is not None else torch.zeros(M, N, device=x.device, dtype=torch.float32)
    ws = _p(workspace) if workspace is not None else None
    nws = workspace.numel() if workspace is not None else 0
    _lib.call("ssm_linear_rows", mode, _p(x), x.stride(0), _p(z) if z is not None else None,
              z.stride(0) if z is not None else 0, _p(g) if g is not None else None, _p(W),
              _p(y), y.stride(0), M, N, K, float(beta), float(eps), ws, nws, _stream())
    return y


def linear(x, W, bias=None, out=None, beta=0.0):
    """y = beta*y + x W^T (+ bias) for any number of rows (ssm_linear, fp32 matrix cores)."""
    M, K = x.shape
    N = W.shape[0]
    y = out if out is not None else torch.zeros(M, N, device=x.device, dtype=torch.float32)
    _lib.call("ssm_linear", _p(x), x.stride(0), _p(W), W.stride(0),
              _p(bias) if bias is not None else None, _p(y), y.stride(0), M, N, K, float(beta),
              _stream())
    return y


def m1_xproj_dt(x, Wx, Wdt, d_state):
    """Mamba-1 x_proj then dt_proj in one pass (ssm_m1_xproj_dt): returns (dbl, dt) with
    dbl = x Wx^T (T, R + 2N) and dt = dbl[:, :R] Wdt^T (T, D)."""
    T, D = x.shape
    R = Wdt.shape[1]
    dbl = torch.empty(T, R + 2 * d_state, device=x.device, dtype=torch.float32)
    dt = torch.empty(T, D, device=x.device, dtype=torch.float32)
    _lib.call("ssm_m1_xproj_dt", _p(x), x.stride(0), _p(Wx), _p(Wdt), _p(dbl), dbl.stride(0),
              _p(dt), dt.stride(0), T, D, R, d_state, _stream())
    return dbl, dt


def gated_rmsnorm(x, z, w, groups=1, eps=1e-5, out=None):
    M, n = x.shape
    y = out if out is not None else torch.empty_like(x)
    _lib.call("ssm_gated_rmsnorm", _p(x), x.stride(0), _p(z), z.stride(0), _p(w), _p(y),
              y.stride(0), M, n, groups, float(eps), _stream())
    return y


# ---------------------------------------------------------------- a linear-attention layer
# Small calls cost what the host spends on them, so each operand is checked with as few calls into
# torch as that takes: contiguous ones (the common case) need no strides.
_CODES = {torch.float32: _lib.SSM_F32, torch.bfloat16: _lib.SSM_BF16}
_f32_t, _i32_t, _i8_t, _f64_t = torch.float32, torch.int32, torch.int8, torch.float64


def _code(dtype):
    code = _CODES.get(dtype)
    if code is None:
        raise TypeError(f"expected float32 or bfloat16, got {dtype}")
    return code


def _here():
    return _device() if _device is not None else torch.cuda.current_device()


def _refuse(name, t, shape, dtype):
    """Why an operand is not of this shape and type on the current device."""
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError("ssmjs_amd kernels need HIP device tensors (no CPU path)")
    raise ValueError(f"{name}: expected a tensor on the current HIP device, got {t.device}")


def _at(name, t, shape, dtype, dev):
    """Device pointer of an operand of this shape and type on device `dev`."""
    if t.dtype != dtype or t.shape != shape or t.get_device() != dev:
        _refuse(name, t, shape, dtype)
    return t.data_ptr()


def _packed(name, t, shape, dtype, dev):
    """_at, of a contiguous operand (None -> NULL)."""
    if t is None:
        return None
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return _at(name, t, shape, dtype, dev)


def _current(name, t):
    """The device of a call: its first operand's, which has to be the current one."""
    if not t.is_cuda:
        raise ValueError("ssmjs_amd kernels need HIP device tensors (no CPU path)")
    dev = t.get_device()
    if dev != _here():
        raise ValueError(f"{name}: expected a tensor on the current HIP device, got {t.device}")
    return dev


def _head_rows(name, t):
    """Row stride of (..., rows, heads, elements): a row's heads follow one another, and the rows
    lie at one distance through all leading dimensions."""
    size = t.shape
    if t.is_contiguous():
        return size[-1] * size[-2]
    st = t.stride()
    if (size[-1] > 1 and st[-1] != 1) or (size[-2] > 1 and st[-2] != size[-1]):
        raise ValueError(f"{name}: the heads of a row must follow one another")
    if len(size) == 3:
        return st[0] if size[0] > 1 else size[1] * size[2]
    ld = st[1] if size[1] > 1 else (st[0] if size[0] > 1 else size[2] * size[3])
    if size[0] > 1 and size[1] > 1 and st[0] != size[1] * ld:
        raise ValueError(f"{name}: rows must lie at one distance")
    return ld


def _ld(name, t):
    """Row stride of a (rows, n) view whose rows are contiguous."""
    if t.is_contiguous():
        return t.shape[1]
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: rows must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def qk_norm_rope(q, k, wq, wk, positions, freqs, eps=1e-6, interleaved=False, out=None):
    """RMS norm of every query and key head with the position rotation (ssm_qk_norm_rope): returns
    (q', k'). q (B,L,H,D) or (B,H,D), k (.., G,D), float32 or bfloat16; wq, wk (D) float32 or None;
    positions int32, the shape of q without its heads; freqs (R/2) float64, radians per position: the
    first R elements of a head turn, in pairs (i, i + R/2) or, interleaved, (2i, 2i + 1); None: norm
    alone. `out`: a pair of tensors, which may be (q, k)."""
    shape, kshape, dt = q.shape, k.shape, q.dtype
    if len(shape) not in (3, 4) or len(kshape) != len(shape):
        raise ValueError("q (B,L,H,D) or (B,H,D), and k of the same rows")
    *rows, H, D = shape
    G = kshape[-2]
    code, dev = _code(dt), _current("q", q)
    T = rows[0] if len(rows) == 1 else rows[0] * rows[1]
    R = 2 * freqs.shape[0] if freqs is not None else 0
    pk = _at("k", k, (*rows, G, D), dt, dev)
    dense = q.is_contiguous() and k.is_contiguous()
    ldq, ldk = (H * D, G * D) if dense else (_head_rows("q", q), _head_rows("k", k))
    if out is None:
        if dense:
            qo, ko = torch.empty_like(q), torch.empty_like(k)
        else:
            qo, ko = q.new_empty(shape), k.new_empty(kshape)
        pqo, pko, ldqo, ldko = qo.data_ptr(), ko.data_ptr(), H * D, G * D
    else:
        qo, ko = out
        pqo, pko = _at("out[0]", qo, shape, dt, dev), _at("out[1]", ko, kshape, dt, dev)
        ldqo, ldko = _head_rows("out[0]", qo), _head_rows("out[1]", ko)
    _lib.call("ssm_qk_norm_rope", code, q.data_ptr(), ldq, pk, ldk,
              _packed("wq", wq, (D,), _f32_t, dev), _packed("wk", wk, (D,), _f32_t, dev),
              _packed("positions", positions, tuple(rows), _i32_t, dev),
              _packed("freqs", freqs, (R // 2,), _f64_t, dev), int(interleaved), eps, pqo, ldqo, pko,
              ldko, T, H, G, D, R, _raw_stream(dev) if _raw_stream is not None else _stream())
    return qo, ko


def linear_attention_workspace(B, L, H, K, V, dtype, device):
    """Workspace for linear_attention (ssm_linear_attention_workspace bytes)."""
    return torch.empty(max(1, _lib.lib().ssm_linear_attention_workspace(_code(dtype), B, L, H, K, V)),
                       dtype=torch.uint8, device=device)


def _own_scratch(workspace, nbytes, t):
    """(tensor, pointer, bytes) of a call's workspace: the caller's, or one for this call."""
    if workspace is not None:
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        if workspace.get_device() != t.get_device():
            raise ValueError(f"workspace: expected a tensor on {t.device}, got {workspace.device}")
        return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()
    if nbytes == 0:
        return None, None, 0
    ws = t.new_empty(nbytes, dtype=torch.uint8)
    return ws, ws.data_ptr(), nbytes


def linear_attention(q, k, v, g, scale=1.0, lengths=None, h0=None, hT=None, out=None,
                     workspace=None):
    """Linear attention with a decay for each head over whole prompts (ssm_linear_attention):
    S_t = e^g S_{t-1} + v_t k_t^T, y_t = scale S_t q_t. q (B,L,H,K), k (B,L,G,K), v (B,L,G,V),
    float32 or bfloat16; g (H) float32; y (B,L,H,V) in their type. lengths (B) int32: rows of y from
    a sequence's length on are zeros, or, in an `out` of the caller's, not written. h0, hT (B,H,V,K) float32, hT may be h0."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q (B,L,H,K), k (B,L,G,K), v (B,L,G,V)")
    B, L, H, K = q.shape
    G, V = k.shape[2], v.shape[3]
    dt = q.dtype
    code, dev = _code(dt), _current("q", q)
    pk, pv = _at("k", k, (B, L, G, K), dt, dev), _at("v", v, (B, L, G, V), dt, dev)
    if out is None:
        out = (q.new_empty if lengths is None else q.new_zeros)((B, L, H, V))
    py = _at("out", out, (B, L, H, V), dt, dev)
    state = (B, H, V, K)
    # (held to the end of the call: freed before, it could be given to another stream)
    ws, pws, nbytes = _own_scratch(
        workspace, _lib.lib().ssm_linear_attention_workspace(code, B, L, H, K, V), q)
    _lib.call("ssm_linear_attention", code, q.data_ptr(), _head_rows("q", q), pk,
              _head_rows("k", k), pv, _head_rows("v", v), _packed("g", g, (H,), _f32_t, dev), scale,
              _packed("lengths", lengths, (B,), _i32_t, dev), py, _head_rows("out", out), B, L, H, G,
              K, V, _packed("h0", h0, state, _f32_t, dev), _packed("hT", hT, state, _f32_t, dev),
              pws, nbytes, _raw_stream(dev) if _raw_stream is not None else _stream())
    return out


def linear_attention_step(q, k, v, g, h, scale=1.0, out=None):
    """One token of linear_attention for every sequence, h (B,H,V,K) float32 in place
    (ssm_linear_attention_step): q (B,H,K), k (B,G,K), v (B,G,V) -> y (B,H,V)."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q (B,H,K), k (B,G,K), v (B,G,V)")
    B, H, K = q.shape
    G, V = k.shape[1], v.shape[2]
    dt = q.dtype
    code, dev = _code(dt), _current("q", q)
    pk, pv = _at("k", k, (B, G, K), dt, dev), _at("v", v, (B, G, V), dt, dev)
    ph = _packed("h", h, (B, H, V, K), _f32_t, dev)
    if ph is None:
        raise ValueError("linear_attention_step needs a state")
    if q.is_contiguous() and k.is_contiguous() and v.is_contiguous():
        ldq, ldk, ldv = H * K, G * K, G * V
    else:
        ldq, ldk, ldv = _head_rows("q", q), _head_rows("k", k), _head_rows("v", v)
    if out is None:
        out = q.new_empty((B, H, V))
        py, ldy = out.data_ptr(), H * V
    else:
        py, ldy = _at("out", out, (B, H, V), dt, dev), _head_rows("out", out)
    _lib.call("ssm_linear_attention_step", code, q.data_ptr(), ldq, pk, ldk, pv, ldv,
              _packed("g", g, (H,), _f32_t, dev), scale, py, ldy, ph, B, H, G, K, V,
              _raw_stream(dev) if _raw_stream is not None else _stream())
    return out


def quantize_rows(x, out=None):
    """Rows of x (M,K), float32 or bfloat16, as 8-bit integers with a scale each
    (ssm_quantize_rows): returns (q (M,K) int8, scale (M) float32). For weights (N,K) this is a scale
    for each output channel."""
    M, K = x.shape
    code, dev = _code(x.dtype), _current("x", x)
    if out is None:
        out = x.new_empty((M, K), dtype=_i8_t), x.new_empty(M, dtype=_f32_t)
    q, scale = out
    _lib.call("ssm_quantize_rows", code, x.data_ptr(), _ld("x", x),
              _at("out[0]", q, (M, K), _i8_t, dev), _ld("out[0]", q),
              _packed("out[1]", scale, (M,), _f32_t, dev), M, K, _stream())
    return q, scale


def _product_out(out, out_dtype, M, N, x, dev):
    """(y, its type's code, pointer, row stride) of a product's outputs."""
    if out is None:
        code = _code(out_dtype)
        out = x.new_empty((M, N), dtype=out_dtype)
        return out, code, out.data_ptr(), N
    return out, _code(out.dtype), _at("out", out, (M, N), out.dtype, dev), _ld("out", out)


def linear_i8(x, sx, W, sw, bias=None, out=None, out_dtype=torch.float32, beta=0.0,
              workspace=None):
    """y = beta*y + sx sw (x W^T) (+ bias) with 8-bit x (M,K) and W (N,K), a scale for each row of
    both (ssm_linear_i8); y in `out_dtype` (or out's), float32 or bfloat16."""
    if out is None and beta != 0:
        raise ValueError("beta needs `out`")
    M, K = x.shape
    N = W.shape[0]
    dev = _current("x", x)
    px, ldx = _at("x", x, (M, K), _i8_t, dev), _ld("x", x)
    pw, ldw = _at("W", W, (N, K), _i8_t, dev), _ld("W", W)
    y, code, py, ldy = _product_out(out, out_dtype, M, N, x, dev)
    ws, pws, nbytes = _own_scratch(
        workspace, _lib.lib().ssm_linear_i8_workspace(px, ldx, pw, ldw, M, N, K), x)
    _lib.call("ssm_linear_i8", px, ldx, _packed("sx", sx, (M,), _f32_t, dev), pw, ldw,
              _packed("sw", sw, (N,), _f32_t, dev), _packed("bias", bias, (N,), _f32_t, dev), code,
              py, ldy, M, N, K, beta, pws, nbytes,
              _raw_stream(dev) if _raw_stream is not None else _stream())
    return y


def linear_q8(x, W, sw, bias=None, out=None, out_dtype=None, beta=0.0, workspace=None):
    """linear_i8 of x (M,K) in float32 or bfloat16, rounded to 8 bits with a scale for each row on
    the way (ssm_linear_q8); y in x's type unless `out_dtype` or `out` say otherwise."""
    if out is None and beta != 0:
        raise ValueError("beta needs `out`")
    M, K = x.shape
    N = W.shape[0]
    dt = x.dtype
    code_x, dev = _code(dt), _current("x", x)
    pw, ldw = _at("W", W, (N, K), _i8_t, dev), _ld("W", W)
    y, code, py, ldy = _product_out(out, out_dtype or dt, M, N, x, dev)
    ws, pws, nbytes = _own_scratch(
        workspace, _lib.lib().ssm_linear_q8_workspace(pw, ldw, M, N, K), x)
    _lib.call("ssm_linear_q8", code_x, x.data_ptr(), _ld("x", x), pw, ldw,
              _packed("sw", sw, (N,), _f32_t, dev), _packed("bias", bias, (N,), _f32_t, dev), code,
              py, ldy, M, N, K, beta, pws, nbytes,
              _raw_stream(dev) if _raw_stream is not None else _stream())
    return y
