"""Host-side operators over the nsosx C ABI (torch supplies device memory and streams).

Each function mirrors the reference operator it replaces (OXN/nsos/ of
vitorGgC569/reimagined): argument meaning, shapes and error behaviour
(ValueError for rejected shapes, as the reference's std::invalid_argument).
All work is enqueued on torch's current stream without synchronising.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from ._lib import NsosxError, call, lib

F32, BF16 = 0, 1
_DT = {torch.float32: F32, torch.bfloat16: BF16}


def _dt(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {t.dtype}: float32 or bfloat16") from None


def _p(t):
    return None if t is None else t.data_ptr()


# torch's current stream handle without a torch.cuda.Stream built around it (1.5 us of host time
# per launch); not part of its public interface
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


def _dev(t: torch.Tensor, name: str, dtype=None) -> torch.Tensor:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    return t


def _opt(t, name: str, dtype=torch.float32):
    return None if t is None else _dev(t, name, dtype)


# ---- weights -------------------------------------------------------------------

def pack_ternary(w) -> tuple[np.ndarray, float]:
    """BitLinear::pack_weights (src/bitlinear.cpp:152-193) on the host.

    w: float [N, K] (numpy or CPU tensor).  Returns (packed uint32 [N*K/16], weight_scale).
    """
    w = np.ascontiguousarray(w.numpy() if isinstance(w, torch.Tensor) else w, dtype=np.float32)
    if w.ndim != 2:
        raise ValueError("pack_ternary expects a 2-D [N, K] matrix")
    n, k = w.shape
    packed = np.zeros(n * k // 16 if k % 16 == 0 else 0, np.uint32)
    ws = ctypes.c_float()
    call("nsosx_pack_ternary", w.ctypes.data_as(ctypes.c_void_p), n, k,
         packed.ctypes.data_as(ctypes.c_void_p), ctypes.byref(ws))
    return packed, float(ws.value)


def unpack_ternary(packed, n: int) -> np.ndarray:
    packed = np.ascontiguousarray(packed, dtype=np.uint32)
    out = np.empty(n, np.int8)
    call("nsosx_unpack_ternary", packed.ctypes.data_as(ctypes.c_void_p), n,
         out.ctypes.data_as(ctypes.c_void_p))
    return out


def find_reserved_code(packed: torch.Tensor, n_codes: int) -> int:
    """Device import check (src/bitlinear.cpp:876-885): index of the first code 3, or -1."""
    _dev(packed, "packed")
    out = torch.empty(1, dtype=torch.int64, device=packed.device)
    call("nsosx_find_reserved_code", _p(packed), n_codes, _p(out), _stream())
    return int(out.item())


def weight_row_sums(packed: torch.Tensor, n: int, k: int) -> torch.Tensor:
    """compute_weight_row_sums (src/bitlinear.cpp:36-73) on the device -> int32 [N]."""
    _dev(packed, "packed")
    if k <= 0 or k % 16 or packed.numel() != n * k // 16:
        raise ValueError("weight_row_sums: packed must hold N*K/16 words with K % 16 == 0")
    out = torch.empty(n, dtype=torch.int32, device=packed.device)
    call("nsosx_weight_row_sums", _p(packed), n, k, _p(out), _stream())
    return out


# ---- BitLinear ------------------------------------------------------------------

def quantize_activations_bitnet(x: torch.Tensor, bits: int = 8, rms_input: bool = False):
    """quantize_activations_bitnet (+ RMS_PERI) -> (q int8 [M,K], act_scale f32 [M])."""
    _dev(x, "x")
    m, k = x.shape
    q = torch.empty((m, k), dtype=torch.int8, device=x.device)
    s = torch.empty(m, dtype=torch.float32, device=x.device)
    ws = torch.empty(m, dtype=torch.float32, device=x.device) if rms_input else None
    call("nsosx_quantize_act_i8", _p(x), _dt(x), m, k, bits, int(rms_input), _p(q), _p(s), _p(ws),
         _stream())
    return q, s


def ternary_gemm(q: torch.Tensor, act_scale: torch.Tensor, packed: torch.Tensor, ws: float,
                 n_out: int, magnitude=None, bias=None, out_dtype=torch.float32,
                 want_acc: bool = False, path: int | None = None, want_y: bool = True):
    """gemm_158bit_i8 integer core + affine (src/bitnet_adapter_avx2.cpp:52-158).

    Returns y [M, N] (or (y, acc int32 [M, N]) with want_acc).
    """
    _dev(q, "q", torch.int8)
    _dev(act_scale, "act_scale", torch.float32)
    _dev(packed, "packed")
    if packed.dtype not in (torch.int32, torch.uint32):
        raise ValueError("packed must hold 32-bit words")
    _opt(magnitude, "magnitude")
    _opt(bias, "bias")
    m, k = q.shape
    y = torch.empty((m, n_out), dtype=out_dtype, device=q.device) if want_y else None
    acc = torch.empty((m, n_out), dtype=torch.int32, device=q.device) if want_acc else None
    ydt = _DT[out_dtype]
    if path is None:
        call("nsosx_ternary_gemm", _p(q), _p(act_scale), _p(packed), ws, m, k, n_out,
             _p(magnitude), _p(bias), _p(y), ydt, _p(acc), _stream())
    else:
        call("nsosx_ternary_gemm_path", _p(q), _p(act_scale), _p(packed), ws, m, k, n_out,
             _p(magnitude), _p(bias), _p(y), ydt, _p(acc), path, _stream())
    if want_acc:
        return y, acc
    return y


# Longest row of the MFMA layout's GEMMs, whose int32 sums are 64 times the ternary ones.
MFMA_LAYOUT_MAX_K = 264208


def skinny_shape(m: int, k: int, n: int) -> bool:
    """The shapes the skinny MFMA decode kernel takes (the library's skinny_ok): 2 <= m <=
    32, k in {1024, 2048, 4096}, ceil(m / 16) * k <= 4096, m * n * 4 < 2^31."""
    return (2 <= m <= 32 and k in (1024, 2048, 4096) and ((m + 15) // 16) * k <= 4096
            and m * n * 4 < 2**31)


def pack_mfma_layout(packed: torch.Tensor) -> torch.Tensor:
    """The prefill GEMM's weight layout (a device repack of reference-layout words)."""
    _dev(packed, "packed")
    out = torch.empty_like(packed)
    call("nsosx_pack_mfma_layout", _p(packed), packed.numel(), _p(out), _stream())
    return out


def ternary_gemm_mfma(q: torch.Tensor, act_scale: torch.Tensor, packed_mfma: torch.Tensor,
                      ws: float, n_out: int, magnitude=None, bias=None,
                      out_dtype=torch.float32, want_acc: bool = False):
    """ternary_gemm on MFMA-layout weights (the prefill MFMA GEMM, K % 128 == 0)."""
    _dev(q, "q", torch.int8)
    _dev(act_scale, "act_scale", torch.float32)
    _dev(packed_mfma, "packed_mfma")
    _opt(magnitude, "magnitude")
    _opt(bias, "bias")
    m, k = q.shape
    y = torch.empty((m, n_out), dtype=out_dtype, device=q.device)
    acc = torch.empty((m, n_out), dtype=torch.int32, device=q.device) if want_acc else None
    call("nsosx_ternary_gemm_mfma", _p(q), _p(act_scale), _p(packed_mfma), ws, m, k, n_out,
         _p(magnitude), _p(bias), _p(y), _DT[out_dtype], _p(acc), _stream())
    return (y, acc) if want_acc else y


def bitnet_gemm_158bit_gpu(x: torch.Tensor, packed: torch.Tensor, weight_scale: float, M: int,
                           K: int, N: int, precision_bits: int = 8, magnitude=None, bias=None,
                           rms_input: bool = False, out_dtype=torch.float32) -> torch.Tensor:
    """bitnet_gemm_158bit_gpu (include/bitnet_gpu_dispatch.h:46-51): quantize + ternary GEMM."""
    _dev(x, "x")
    _dev(packed, "packed")
    if x.numel() != M * K:
        raise ValueError("bitnet_gemm_158bit_gpu: x does not hold M*K elements")
    qw = torch.empty((M, K), dtype=torch.int8, device=x.device)
    sw = torch.empty(M, dtype=torch.float32, device=x.device)
    rw = torch.empty(M, dtype=torch.float32, device=x.device) if rms_input else None
    y = torch.empty((M, N), dtype=out_dtype, device=x.device)
    call("nsosx_bitlinear_forward", _p(x), _dt(x), _p(packed), weight_scale, M, K, N,
         precision_bits, int(rms_input), _p(magnitude), _p(bias), _p(y), _DT[out_dtype], _p(qw),
         _p(sw), _p(rw), _stream())
    return y


def linear_f32(x: torch.Tensor, w: torch.Tensor, rms_input: bool = False, magnitude=None,
               bias=None, out_dtype=torch.float32, out=None) -> torch.Tensor:
    """BitLinear's float reference path for quantization-sensitive layers
    (src/bitlinear.cpp:465-518): [rmsnorm] x @ w^T, then * magnitude, then + bias."""
    _dev(x, "x")
    _dev(w, "w", torch.float32)
    _opt(magnitude, "magnitude")
    _opt(bias, "bias")
    if x.dim() != 2 or w.dim() != 2 or w.shape[1] != x.shape[1]:
        raise ValueError("linear_f32: x [M, K] and w [N, K] must agree in K")
    m, k = x.shape
    n = w.shape[0]
    for name, v in (("magnitude", magnitude), ("bias", bias)):
        if v is not None and v.numel() != n:
            raise ValueError(f"linear_f32: {name} must hold N = {n} values")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=x.device)
    elif tuple(out.shape) != (m, n) or not out.is_contiguous():
        raise ValueError("linear_f32: out must be a contiguous [M, N] tensor")
    rw = torch.empty(m, dtype=torch.float32, device=x.device) if rms_input else None
    call("nsosx_linear_f32", _p(x), _dt(x), m, k, _p(w), n, int(rms_input), _p(magnitude),
         _p(bias), _p(out), _dt(out), _p(rw), _stream())
    return out


def bitlinear_ste_backward(x, q, act_scale, w_latent, packed, weight_scale: float, grad,
                           rms_input: bool = True, magnitude=None, want_dbias: bool = False,
                           want_dmag: bool = True) -> dict:
    """BitLinear::backward on the packed path (src/bitlinear.cpp:1191-1357) from what the
    forward saved: x [M, K], its int8 codes q and act_scale, the latent weights [N, K] and
    their packed ternary; grad [M, N].  Returns dx, dW (+ dmag, dbias)."""
    for name, v, dt in (("q", q, torch.int8), ("act_scale", act_scale, torch.float32),
                        ("w_latent", w_latent, torch.float32), ("grad", grad, torch.float32)):
        _dev(v, name, dt)
    _dev(packed, "packed")
    _opt(magnitude, "magnitude")
    m, k = q.shape
    n = w_latent.shape[0]
    if tuple(grad.shape) != (m, n) or tuple(w_latent.shape) != (n, k) or \
            act_scale.numel() != m or packed.numel() != n * k // 16:
        raise ValueError("bitlinear_ste_backward: inconsistent shapes")
    if rms_input:
        _dev(x, "x")
        if tuple(x.shape) != (m, k):
            raise ValueError("bitlinear_ste_backward: x must be [M, K]")
    dev = q.device
    out = {"dx": torch.empty((m, k), dtype=torch.float32, device=dev),
           "dW": torch.empty((n, k), dtype=torch.float32, device=dev)}
    if magnitude is not None and want_dmag:
        out["dmag"] = torch.empty(n, dtype=torch.float32, device=dev)
    if want_dbias:
        out["dbias"] = torch.empty(n, dtype=torch.float32, device=dev)
    nbytes = int(lib().nsosx_bitlinear_ste_backward_workspace(m, k, n, int(rms_input)))
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
    call("nsosx_bitlinear_ste_backward", _p(x) if rms_input else None,
         _dt(x) if rms_input else F32, _p(q), _p(act_scale), _p(w_latent), _p(packed),
         float(weight_scale), m, k, n, int(rms_input), _p(magnitude), _p(grad), _p(out["dx"]),
         _p(out["dW"]), _p(out.get("dmag")), _p(out.get("dbias")), _p(ws), _stream())
    return out


class LinearViewArray:
    """Device array of nsosx_linear_view descriptors (GpuLinearView's C shape).

    Borrows the tensors it points at; keeps Python references so they outlive it.
    """

    class _View(ctypes.Structure):
        _fields_ = [("packed", ctypes.c_void_p), ("magnitude", ctypes.c_void_p),
                    ("bias", ctypes.c_void_p), ("inputs", ctypes.c_int),
                    ("outputs", ctypes.c_int), ("weight_scale", ctypes.c_float)]

    def __init__(self, entries, device):
        self._keep = []
        arr = (self._View * len(entries))()
        for i, (packed, ws, inputs, outputs, mag, bias) in enumerate(entries):
            self._keep += [packed, mag, bias]
            arr[i].packed = packed.data_ptr()
            arr[i].magnitude = None if mag is None else mag.data_ptr()
            arr[i].bias = None if bias is None else bias.data_ptr()
            arr[i].inputs = inputs
            arr[i].outputs = outputs
            arr[i].weight_scale = ws
        raw = bytes(arr)
        host = torch.frombuffer(bytearray(raw), dtype=torch.uint8)
        self.tensor = host.to(device)
        self.count = len(entries)

    @property
    def ptr(self):
        return self.tensor.data_ptr()


class DecodeViewArray:
    """Device array of nsosx_decode_view descriptors (GpuLinearView, include/gpu_linear_view.h:8-25):
    entries are dicts with either `packed` (int32 words) + `weight_scale` + `bits`, or `weight`
    (f32 [outputs, inputs]); `inputs`, `outputs`, optional `magnitude`, `bias`, `rms_input`."""

    class _View(ctypes.Structure):
        _fields_ = [("weight", ctypes.c_void_p), ("packed", ctypes.c_void_p),
                    ("magnitude", ctypes.c_void_p), ("bias", ctypes.c_void_p),
                    ("inputs", ctypes.c_int), ("outputs", ctypes.c_int),
                    ("activation_bits", ctypes.c_int), ("rms_input", ctypes.c_int),
                    ("weight_scale", ctypes.c_float)]

    def __init__(self, entries, device):
        self._keep = []
        arr = (self._View * len(entries))()
        for i, e in enumerate(entries):
            ptr = lambda t: None if t is None else t.data_ptr()
            for k in ("weight", "packed", "magnitude", "bias"):
                if e.get(k) is not None:
                    self._keep.append(e[k])
            arr[i].weight = ptr(e.get("weight"))
            arr[i].packed = ptr(e.get("packed"))
            arr[i].magnitude = ptr(e.get("magnitude"))
            arr[i].bias = ptr(e.get("bias"))
            arr[i].inputs = int(e["inputs"])
            arr[i].outputs = int(e["outputs"])
            arr[i].activation_bits = int(e.get("bits", 0 if e.get("packed") is None else 8))
            arr[i].rms_input = int(bool(e.get("rms_input", False)))
            arr[i].weight_scale = float(e.get("weight_scale", 1.0))
        self.tensor = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).to(device)
        self.count = len(entries)
        self.max_outputs = max(int(e["outputs"]) for e in entries)

    @property
    def ptr(self):
        return self.tensor.data_ptr()


def grouped_decode_projections(views: DecodeViewArray, x: torch.Tensor, out_dtype=None,
                               out=None) -> torch.Tensor:
    """GpuProjectionGroup::forward (src/gpu_projection_group.cpp:12-49): one input row
    through every view -> [views, max outputs] (row g holds view g's outputs first)."""
    _dev(x, "x")
    if x.dim() != 1 and not (x.dim() == 2 and x.shape[0] == 1):
        raise ValueError("grouped_decode_projections: x must be one row")
    odt = out_dtype or x.dtype
    if out is None:
        out = torch.empty((views.count, views.max_outputs), dtype=odt, device=x.device)
    elif tuple(out.shape) != (views.count, views.max_outputs) or not out.is_contiguous():
        raise ValueError("grouped_decode_projections: out must be [views, max outputs]")
    call("nsosx_grouped_decode_projections", views.ptr, views.count, _p(x), _dt(x), _p(out),
         views.max_outputs, _dt(out), _stream())
    return out


def grouped_gemv(views: LinearViewArray, q: torch.Tensor, act_scale: torch.Tensor, n_out: int,
                 out_dtype=torch.bfloat16) -> torch.Tensor:
    """Grouped decode projections (include/cuda/kernels.cuh:27-29).

    q: int8 [G, M, K]; act_scale [G, M]; returns y [G, M, n_out].
    """
    g, m, k = q.shape
    y = torch.empty((g, m, n_out), dtype=out_dtype, device=q.device)
    call("nsosx_grouped_gemv", views.ptr, g, _p(q), m * k, _p(act_scale), m, m, _p(y), m * n_out,
         _DT[out_dtype], _stream())
    return y


# ---- Mamba ----------------------------------------------------------------------

def _shape(t, want: tuple, name: str, fn: str) -> None:
    if t is not None and t.shape != tuple(want):
        raise ValueError(f"{fn}: {name} must have shape {tuple(want)}, got {tuple(t.shape)}")


def _check_scan_shapes(fn, x, dt, a_log, B, C, D, z, H, P, N, G, t_rows=None):
    """Host-side shape checks of the scan inputs: the C ABI takes raw pointers, so an
    undersized buffer would be read or written out of bounds on the device."""
    if min(H, P, N, G) <= 0 or H % G:
        raise ValueError(f"{fn}: need positive H, P, N, G with G dividing H")
    if x.dim() != 2 or x.shape[1] != H * P:
        raise ValueError(f"{fn}: x must be [T, H*P] = [T, {H * P}], got {tuple(x.shape)}")
    t = x.shape[0] if t_rows is None else t_rows
    _shape(dt, (t, H), "dt", fn)
    _shape(B, (t, G * N), "B", fn)
    _shape(C, (t, G * N), "C", fn)
    _shape(z, (t, H * P), "z", fn)
    if D.numel() != H:
        raise ValueError(f"{fn}: D must hold H = {H} values, got {D.numel()}")
    if a_log.numel() not in (H, H * N):
        raise ValueError(f"{fn}: a_log must hold H or H*N values, got {a_log.numel()}")


def _check_cu_seqlens(fn, cu_seqlens):
    """Offsets outside [0, T] are clamped by the kernels; the count must be S+1 >= 2."""
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
        raise ValueError(f"{fn}: cu_seqlens must be a 1-D int32 tensor of S+1 >= 2 offsets")


def conv1d_causal(x: torch.Tensor, weight: torch.Tensor, cu_seqlens: torch.Tensor, bias=None,
                  silu: bool = True, out_dtype=None) -> torch.Tensor:
    """Depthwise causal conv + bias + SiLU per sequence (src/mamba2.cpp:1056-1076, 2437-2446).

    x may be a column slice of a wider row-major tensor (unit stride in the last dim).
    """
    if x.stride(1) != 1:
        raise ValueError("conv1d_causal: x must have unit stride in the channel dim")
    _dev(weight, "weight", torch.float32)
    _dev(cu_seqlens, "cu_seqlens", torch.int32)
    _opt(bias, "bias")
    t, c = x.shape
    out_dtype = out_dtype or x.dtype
    out = torch.empty((t, c), dtype=out_dtype, device=x.device)
    call("nsosx_conv1d_causal", _p(x), _dt(x), x.stride(0), _p(weight), _p(bias), _p(cu_seqlens),
         cu_seqlens.numel() - 1, t, c, weight.shape[1], int(silu), _p(out), _DT[out_dtype],
         _stream())
    return out


def _scan_workspace(s, t, H, P, N, chunk_tokens, device):
    nbytes = int(lib().nsosx_scan_fwd_workspace(s, t, H, P, N, chunk_tokens))
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)


def selective_scan_fwd(x, dt, a_log, B, C, D, z, cu_seqlens, H, P, N, G, initial_state=None,
                       want_final: bool = True, chunk_tokens: int | None = -1):
    """Packed ragged faithful scan (src/mamba2.cpp:2602-2675) -> (y [T, H*P], final [S, H*P, N]).

    chunk_tokens: -1 lets the library chunk long sequences in time when the batch cannot
    fill the GPU, 0 never chunks, > 0 forces that chunk length; None calls the unplanned
    entry point (no order pre-pass, no chunking)."""
    _check_scan_shapes("selective_scan_fwd", x, dt, a_log, B, C, D, z, H, P, N, G)
    _check_cu_seqlens("selective_scan_fwd", cu_seqlens)
    t = x.shape[0]
    s = cu_seqlens.numel() - 1
    _shape(initial_state, (s, H * P, N), "initial_state", "selective_scan_fwd")
    if not x.is_cuda:
        raise ValueError("x must be a device tensor")
    if x.stride(1) != 1 or (z is not None and z.stride(1) != 1):
        raise ValueError("selective_scan_fwd: x and z need unit stride in the channel dim")
    for name, v in (("dt", dt), ("B", B), ("C", C)):
        _dev(v, name, x.dtype)
    if z is not None and z.dtype != x.dtype:
        raise ValueError("selective_scan_fwd: z must have x's dtype")
    _dev(a_log, "a_log", torch.float32)
    _dev(D, "D", torch.float32)
    _dev(cu_seqlens, "cu_seqlens", torch.int32)
    _opt(initial_state, "initial_state")
    a_per_state = int(a_log.numel() == H * N and N > 1)
    y = torch.empty((t, H * P), dtype=x.dtype, device=x.device)
    fin = torch.empty((s, H * P, N), dtype=torch.float32, device=x.device) if want_final else None
    if chunk_tokens is None:
        call("nsosx_selective_scan_fwd", _p(x), x.stride(0), _p(dt), _p(a_log), a_per_state,
             _p(B), _p(C), _p(D), _p(z), 0 if z is None else z.stride(0), _p(cu_seqlens), s, t,
             H, P, N, G, _dt(x), _p(initial_state), _p(fin), _p(y), _stream())
    else:
        ws = _scan_workspace(s, t, H, P, N, chunk_tokens, x.device)
        call("nsosx_scan_fwd_planned", _p(x), x.stride(0), None, None, 0, _p(dt), _p(a_log),
             a_per_state, _p(B), _p(C), _p(D), _p(z), 0 if z is None else z.stride(0),
             _p(cu_seqlens), s, t, H, P, N, G, _dt(x), _p(initial_state), _p(fin), _p(y),
             chunk_tokens, _p(ws), _stream())
    return y, fin


def conv_scan_fwd(x_raw, conv_w, conv_b, dt, a_log, B, C, D, z, cu_seqlens, H, P, N, G,
                  initial_state=None, want_final: bool = True, chunk_tokens: int | None = -1):
    """Causal conv + bias + SiLU fused into the scan's staging -> (y, final state).
    chunk_tokens as selective_scan_fwd."""
    _check_scan_shapes("conv_scan_fwd", x_raw, dt, a_log, B, C, D, z, H, P, N, G)
    _check_cu_seqlens("conv_scan_fwd", cu_seqlens)
    t = x_raw.shape[0]
    s = cu_seqlens.numel() - 1
    _shape(initial_state, (s, H * P, N), "initial_state", "conv_scan_fwd")
    if conv_w.dim() != 2 or conv_w.shape[0] != H * P or not 1 <= conv_w.shape[1] <= 8:
        raise ValueError(f"conv_scan_fwd: conv_w must be [H*P, W] = [{H * P}, 1..8], "
                         f"got {tuple(conv_w.shape)}")
    if conv_b is not None and conv_b.numel() != H * P:
        raise ValueError(f"conv_scan_fwd: conv_b must hold H*P = {H * P} values")
    if not x_raw.is_cuda:
        raise ValueError("x_raw must be a device tensor")
    if x_raw.stride(1) != 1 or (z is not None and z.stride(1) != 1):
        raise ValueError("conv_scan_fwd: x and z need unit stride in the channel dim")
    for name, v in (("dt", dt), ("B", B), ("C", C)):
        _dev(v, name, x_raw.dtype)
    _dev(conv_w, "conv_w", torch.float32)
    _opt(conv_b, "conv_b")
    _dev(a_log, "a_log", torch.float32)
    _dev(D, "D", torch.float32)
    _dev(cu_seqlens, "cu_seqlens", torch.int32)
    _opt(initial_state, "initial_state")
    a_per_state = int(a_log.numel() == H * N and N > 1)
    y = torch.empty((t, H * P), dtype=x_raw.dtype, device=x_raw.device)
    fin = (torch.empty((s, H * P, N), dtype=torch.float32, device=x_raw.device)
           if want_final else None)
    if chunk_tokens is None:
        call("nsosx_conv_scan_fwd", _p(x_raw), x_raw.stride(0), _p(conv_w), _p(conv_b),
             conv_w.shape[1], _p(dt), _p(a_log), a_per_state, _p(B), _p(C), _p(D), _p(z),
             0 if z is None else z.stride(0), _p(cu_seqlens), s, t, H, P, N, G, _dt(x_raw),
             _p(initial_state), _p(fin), _p(y), _stream())
    else:
        ws = _scan_workspace(s, t, H, P, N, chunk_tokens, x_raw.device)
        call("nsosx_scan_fwd_planned", _p(x_raw), x_raw.stride(0), _p(conv_w), _p(conv_b),
             conv_w.shape[1], _p(dt), _p(a_log), a_per_state, _p(B), _p(C), _p(D), _p(z),
             0 if z is None else z.stride(0), _p(cu_seqlens), s, t, H, P, N, G, _dt(x_raw),
             _p(initial_state), _p(fin), _p(y), chunk_tokens, _p(ws), _stream())
    return y, fin


def selective_scan_step(x, dt, a_log, B, C, D, z, state, H, P, N, G):
    """Decode step in place on `state` [R, H*P, N] (src/mamba2.cpp:4038-4125) -> y [R, H*P]."""
    _check_scan_shapes("selective_scan_step", x, dt, a_log, B, C, D, z, H, P, N, G)
    r = x.shape[0]
    _shape(state, (r, H * P, N), "state", "selective_scan_step")
    for name, v in (("x", x), ("dt", dt), ("B", B), ("C", C)):
        _dev(v, name, x.dtype)
    if z is not None:
        _dev(z, "z", x.dtype)
    _dev(a_log, "a_log", torch.float32)
    _dev(D, "D", torch.float32)
    _dev(state, "state", torch.float32)
    a_per_state = int(a_log.numel() == H * N and N > 1)
    y = torch.empty_like(x)
    call("nsosx_selective_scan_step", _p(x), _p(dt), _p(a_log), a_per_state, _p(B), _p(C), _p(D),
         _p(z), r, H, P, N, G, _dt(x), _p(state), _p(y), _stream())
    return y


def _mamba2_step_width(conv_w, conv_b, ring, a_log, D, norm_w, state, r, inner, gs, H, N) -> int:
    """Checks mamba2_step's weights and states; returns the conv width."""
    cd = inner + 2 * gs
    _dev(conv_w, "conv_w", torch.float32)
    width = conv_w.shape[1]
    for name, t, want in (("conv_w", conv_w, (cd, width)), ("conv_b", conv_b, (cd,)),
                          ("ring", ring if width > 1 else None, (r, width - 1, cd)),
                          ("a_log", a_log, (H,)), ("D", D, (H,)), ("norm_w", norm_w, (inner,)),
                          ("state", state, (r, inner, N))):
        if t is None and (name in ("conv_b", "norm_w") or (name == "ring" and width <= 1)):
            continue
        # (one line where all is well: a decode step runs this on every call)
        if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous() and t.shape == want):
            _shape(_dev(t, name, torch.float32), want, name, "mamba2_step")
    return width


def _mamba2_step_out_proj(packed, mag, bias, d, inner) -> None:
    _dev(packed, "out_proj packed")
    if packed.numel() != d * inner // 16:
        raise ValueError("mamba2_step: out_proj weights must be [d, H*P/16] words and out [R, d]")
    _opt(mag, "out_proj magnitude")
    _opt(bias, "out_proj bias")


def mamba2_step(x, z, B, C, dt, conv_w, conv_b, ring, a_log, D, norm_w, state, H, P, N, G,
                eps: float = 1e-5, act_bits: int = 8, q=None, act_scale=None, y=None,
                out_proj=None, out=None):
    """The faithful Mamba-2 decode step after its projections, one launch
    (src/mamba2.cpp:4038-4125 through out_proj's input quantization, src/bitlinear.cpp:240-291):
    the conv ring over x | B | C, the state step, RMSNorm(y * SiLU(z)) * norm_w and its int8
    codes, in place on `ring` [R, W-1, H*P + 2*G*N] and `state` [R, H*P, N].

    x, z [R, H*P]; B, C [R, G*N] and dt [R, H] (bias included): column slices of one
    projection output sharing its row stride.  -> (q int8 [R, H*P], act_scale f32 [R],
    y [R, H*P] the pre-gate output).

    out_proj: (packed int32 words [d, H*P / 16], weight_scale, magnitude, bias) of the
    block's ternary out_proj; with it and `out` [R, d] the step also runs the out_proj
    on the codes (nsosx_mamba2_step_out: one launch fewer at one row)."""
    inner, gs = H * P, G * N
    r = x.shape[0]
    _dev(x, "x")
    _dev(z, "z", x.dtype)
    _shape(x, (r, inner), "x", "mamba2_step")
    _shape(z, (r, inner), "z", "mamba2_step")
    stride = B.stride(0) if r > 1 else max(B.stride(0), C.stride(0), dt.stride(0))
    for name, v, n in (("B", B, gs), ("C", C, gs), ("dt", dt, H)):
        if not v.is_cuda or v.dtype != x.dtype or tuple(v.shape) != (r, n) or v.stride(1) != 1:
            raise ValueError(f"mamba2_step: {name} must be a device [{r}, {n}] {x.dtype} view "
                             "with unit column stride")
        if r > 1 and v.stride(0) != stride:
            raise ValueError("mamba2_step: B, C and dt must share one row stride")
    width = _mamba2_step_width(conv_w, conv_b, ring, a_log, D, norm_w, state, r, inner, gs, H, N)
    if q is None:
        q = torch.empty((r, inner), dtype=torch.int8, device=x.device)
    if act_scale is None:
        act_scale = torch.empty(r, dtype=torch.float32, device=x.device)
    _shape(_dev(q, "q", torch.int8), (r, inner), "q", "mamba2_step")
    _shape(_dev(act_scale, "act_scale", torch.float32), (r,), "act_scale", "mamba2_step")
    if y is None:
        y = torch.empty_like(x)
    _shape(_dev(y, "y", x.dtype), (r, inner), "y", "mamba2_step")
    args = (_p(x), _p(z), _p(B), _p(C), _p(dt), stride, _p(conv_w), _p(conv_b), width,
            _p(ring) if width > 1 else None, _p(a_log), _p(D), _p(norm_w), eps, r, H, P, N, G,
            _dt(x), _p(state), _p(y), _p(q), _p(act_scale), act_bits)
    if out_proj is None:
        call("nsosx_mamba2_step", *args, _stream())
        return q, act_scale, y
    packed, ws, mag, bias = out_proj
    d = out.shape[1]
    if tuple(out.shape) != (r, d) or not out.is_contiguous():
        raise ValueError("mamba2_step: out_proj weights must be [d, H*P/16] words and out [R, d]")
    _mamba2_step_out_proj(packed, mag, bias, d, inner)
    call("nsosx_mamba2_step_out", *args, _p(packed), ws, d, _p(mag), _p(bias), _p(out), _dt(out),
         _stream())
    return q, act_scale, y


# ---- MoE ------------------------------------------------------------------------

def valid_rows_mask(valid_rows, rows: int, device) -> torch.Tensor | None:
    """The reference's 0/1 valid-row mask on the device (None: every row valid).  A host
    mask is checked as MoERouter::forward checks it (src/jamba.cpp:8145-8153): one entry
    per row, each 0 or 1, else ValueError; a uint8 device tensor is taken as is (the
    routing then treats any nonzero byte as valid, as the reference's device kernel
    does)."""
    if valid_rows is None:
        return None
    if isinstance(valid_rows, torch.Tensor) and valid_rows.is_cuda:
        if valid_rows.dtype != torch.uint8 or valid_rows.numel() != rows:
            raise ValueError("MoERouter valid-row mask size mismatch")
        return valid_rows.contiguous()
    v = np.asarray(valid_rows.cpu() if isinstance(valid_rows, torch.Tensor) else valid_rows)
    if v.size == 0:
        return None
    if v.size != rows:
        raise ValueError("MoERouter valid-row mask size mismatch")
    if np.any((v != 0) & (v != 1)):
        raise ValueError("MoERouter valid-row mask must contain only 0 or 1")
    return torch.from_numpy(v.astype(np.uint8).reshape(-1)).to(device)


def moe_route(logits: torch.Tensor, k: int = 2, select_only: bool = False, valid_rows=None,
              want_loads: bool = False) -> dict:
    """MoERouter::forward(x, valid_rows) from logits + forward_moe's ordered dispatch, on the
    device.  select_only: weights and selected only (one launch), as the sparse decode needs.
    valid_rows: the reference's 0/1 padding mask (host array or uint8 device tensor), None
    for every row valid; padding rows get zero weights, selections -1 and no slots.
    want_loads: also "loads", the per-expert sums of the weights (expert_loads)."""
    _dev(logits, "logits", torch.float32)
    rows, e = logits.shape
    dev = logits.device
    mask = valid_rows_mask(valid_rows, rows, dev)
    out = {
        "weights": torch.empty((rows, e), dtype=torch.float32, device=dev),
        "selected": torch.empty((rows, k), dtype=torch.int32, device=dev),
    }
    if want_loads:
        out["loads"] = torch.empty(e, dtype=torch.float32, device=dev)
    loads = _p(out["loads"]) if want_loads else None
    if select_only:
        call("nsosx_moe_route", _p(logits), _p(mask), rows, e, k, _p(out["weights"]),
             _p(out["selected"]), None, None, None, None, loads, None, _stream())
        return out
    out.update({
        "counts": torch.empty(e, dtype=torch.int32, device=dev),
        "offsets": torch.empty(e + 1, dtype=torch.int32, device=dev),
        "perm": torch.empty(rows * k, dtype=torch.int32, device=dev),
        "slot_of": torch.empty((rows, k), dtype=torch.int32, device=dev),
    })
    ws = torch.empty(max(1, int(lib().nsosx_moe_route_workspace(rows, e))), dtype=torch.int32,
                     device=dev)
    call("nsosx_moe_route", _p(logits), _p(mask), rows, e, k, _p(out["weights"]),
         _p(out["selected"]), _p(out["counts"]), _p(out["offsets"]), _p(out["perm"]),
         _p(out["slot_of"]), loads, _p(ws), _stream())
    return out


def grouped_ternary_gemm(views: LinearViewArray, offsets, perm, q, act_scale, n_out: int,
                         max_rows_per_expert: int, squared_relu: bool = False,
                         gather: bool = True, out_dtype=torch.float32,
                         total_rows: int | None = None) -> torch.Tensor:
    """Per-expert ternary GEMMs over slot segments -> y [slots, n_out] in slot order.

    total_rows: an upper bound on offsets[E] (default: the slot count) so the launch covers
    only the real row tiles; 0 launches max_rows_per_expert rows of tiles per expert."""
    _dev(offsets, "offsets", torch.int32)
    if gather:
        _dev(perm, "perm", torch.int32)
    _dev(q, "q", torch.int8)
    _dev(act_scale, "act_scale", torch.float32)
    slots = int(perm.numel()) if gather else q.shape[0]
    k = q.shape[1]
    y = torch.empty((slots, n_out), dtype=out_dtype, device=q.device)
    total = slots if total_rows is None else int(total_rows)
    call("nsosx_grouped_ternary_gemm", views.ptr, views.count, _p(offsets), _p(perm), int(gather),
         _p(q), _p(act_scale), k, n_out, max_rows_per_expert, total, int(squared_relu), _p(y),
         _DT[out_dtype], _stream())
    return y


def grouped_ternary_gemm_mfma(views: LinearViewArray, offsets, perm, q, act_scale, n_out: int,
                              total_rows: int, squared_relu: bool = False, gather: bool = True,
                              out_dtype=torch.float32, workspace=None) -> torch.Tensor:
    """grouped_ternary_gemm on views holding MFMA-layout weights (compact row tiles).  With a
    workspace (uint8 device tensor of grouped_mfma_workspace_bytes()), the entry that splits a
    sparse last round of tiles along K (nsosx_grouped_ternary_gemm_mfma_ws; same bits)."""
    _dev(offsets, "offsets", torch.int32)
    if gather:
        _dev(perm, "perm", torch.int32)
    _dev(q, "q", torch.int8)
    _dev(act_scale, "act_scale", torch.float32)
    slots = int(perm.numel()) if gather else q.shape[0]
    k = q.shape[1]
    y = torch.empty((slots, n_out), dtype=out_dtype, device=q.device)
    if workspace is None:
        call("nsosx_grouped_ternary_gemm_mfma", views.ptr, views.count, _p(offsets), _p(perm),
             int(gather), _p(q), _p(act_scale), k, n_out, int(total_rows), int(squared_relu),
             _p(y), _DT[out_dtype], _stream())
    else:
        _dev(workspace, "workspace", torch.uint8)
        call("nsosx_grouped_ternary_gemm_mfma_ws", views.ptr, views.count, _p(offsets), _p(perm),
             int(gather), _p(q), _p(act_scale), k, n_out, int(total_rows), int(squared_relu),
             _p(y), _DT[out_dtype], _p(workspace), int(workspace.numel()), _stream())
    return y


def grouped_mfma_workspace_bytes() -> int:
    """Bytes of the split-K tail workspace of nsosx_grouped_ternary_gemm_mfma_ws on the current
    device (2 x CUs x 128 KiB)."""
    n = int(lib().nsosx_grouped_ternary_gemm_mfma_workspace())
    if n <= 0:
        raise NsosxError("nsosx_grouped_ternary_gemm_mfma_workspace", n, "no device")
    return n


def moe_combine(expert_out, slot_of, selected, weights, out_dtype=torch.float32) -> torch.Tensor:
    _dev(slot_of, "slot_of", torch.int32)
    _dev(selected, "selected", torch.int32)
    _dev(weights, "weights", torch.float32)
    rows, e = weights.shape
    k = selected.shape[1]
    dim = expert_out.shape[1]
    out = torch.empty((rows, dim), dtype=out_dtype, device=expert_out.device)
    call("nsosx_moe_combine", _p(expert_out), _dt(expert_out), _p(slot_of), _p(selected),
         _p(weights), rows, e, k, dim, _p(out), _DT[out_dtype], _stream())
    return out


# ---- scored routing and int8 experts ----------------------------------------------

_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _on(fn: str, dev: int, *tensors) -> None:
    """Checks (name, tensor or None, dtype or None, shape or None) each: contiguous tensors of
    device `dev`, which has to be the current one (whose stream the call goes to)."""
    for name, t, dtype, shape in tensors:
        # (one line where all is well: a decode step runs this on every call)
        if t is None or (t.get_device() == dev >= 0 and t.is_contiguous() and
                         (dtype is None or t.dtype == dtype) and
                         (shape is None or t.shape == shape)):
            continue
        _dev(t, name, dtype)
        if t.get_device() != dev:
            raise ValueError(f"{fn}: {name} must be on device {dev}, got {t.device}")
        raise ValueError(f"{fn}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if _current_device() != dev:
        raise ValueError(f"{fn}: the tensors' device {dev} must be the current one")


def _stream_on(dev: int):
    return _stream() if _raw_stream is None else _raw_stream(dev)


def _too_many(fn: str, name: str, shape) -> ValueError:
    """For sizes that the C entries' int cannot hold (ctypes would pass their lowest 32 bits)."""
    return ValueError(f"{fn}: {name} must have less than 2^31 rows and columns, got {tuple(shape)}")


def _logit_rows(fn: str, logits: torch.Tensor) -> int:
    """Checks router logits [rows, E] (a column slice of a wider tensor is fine); row stride."""
    shape = logits.shape
    if len(shape) == 2 and (shape[0] | shape[1]) >> 31:
        raise _too_many(fn, "logits", shape)
    if not logits.is_cuda:
        raise ValueError("logits must be a device tensor")
    if len(shape) != 2 or 0 in shape:
        raise ValueError(f"{fn}: logits must be [rows, experts], got {tuple(shape)}")
    _dt(logits)
    rows, e = shape
    if (e > 1 and logits.stride(1) != 1) or (rows > 1 and logits.stride(0) < e):
        raise ValueError(f"{fn}: logits need unit column stride and rows that do not overlap")
    return logits.stride(0) if rows > 1 else e


def _score_mode(fn: str, score: str) -> int:
    if score not in ("softmax", "sigmoid"):
        raise ValueError(f"{fn}: score must be 'softmax' or 'sigmoid', got {score!r}")
    return int(score == "sigmoid")


def moe_route_scored(logits: torch.Tensor, k: int, score: str = "softmax", bias=None,
                     groups: int = 1, group_keep: int | None = None, group_best: int = 2,
                     renorm: bool = True, scale: float = 1.0, valid_rows=None,
                     select_only: bool = False) -> dict:
    """Routing by softmax or sigmoid scores, with a balance bias [E] that takes part in the
    choice only, group-limited choice (the group_keep best of `groups` equal runs of experts by
    the sum of their group_best largest values), top-k <= 16 of up to 512 experts and weights
    renormalised over the choice and scaled (nsosx_moe_route_scored).

    logits f32 or bf16 [rows, E].  -> weights f32 [rows, k], selected int32 [rows, k], and,
    unless select_only, counts [E], offsets [E+1], perm [rows*k] (-1 past offsets[E]) and
    slot_of [rows, k] for grouped_int8_gemm and moe_combine_topk.  valid_rows as moe_route.
    No autograd: the results are detached, moe_route_scored_backward gives the logits' gradient."""
    fn = "moe_route_scored"
    stride = _logit_rows(fn, logits)
    rows, e = logits.shape
    sig = _score_mode(fn, score)
    dev = logits.device
    mask = valid_rows_mask(valid_rows, rows, dev)
    _on(fn, logits.get_device(), ("bias", bias, torch.float32, (e,)),
        ("valid_rows", mask, torch.uint8, None))
    if not 0 < k <= e:
        raise ValueError(f"{fn}: need 0 < k <= {e} experts, got {k}")
    keep = groups if group_keep is None else group_keep
    # the int32 outputs (and the workspace behind them) are pieces of one buffer
    n = rows * k
    w = torch.empty((rows, k), dtype=torch.float32, device=dev)
    if select_only:
        sel = torch.empty((rows, k), dtype=torch.int32, device=dev)
        call("nsosx_moe_route_scored", _p(logits), _dt(logits), stride, _p(mask), _p(bias), rows, e,
             k, sig, groups, keep, group_best, int(renorm), float(scale), _p(w), _p(sel), None,
             None, None, None, None, _stream_on(logits.get_device()))
        return {"weights": w, "selected": sel}
    ws = max(1, int(lib().nsosx_moe_route_scored_workspace(rows, e)))
    buf = torch.empty(3 * n + 2 * e + 1 + ws, dtype=torch.int32, device=dev)
    sel, slot_of, perm, counts, offsets, ws = buf.split((n, n, n, e, e + 1, ws))
    sel, slot_of = sel.view(rows, k), slot_of.view(rows, k)
    call("nsosx_moe_route_scored", _p(logits), _dt(logits), stride, _p(mask), _p(bias), rows, e, k,
         sig, groups, keep, group_best, int(renorm), float(scale), _p(w), _p(sel), _p(counts),
         _p(offsets), _p(perm), _p(slot_of), _p(ws), _stream_on(logits.get_device()))
    return {"weights": w, "selected": sel, "counts": counts, "offsets": offsets, "perm": perm,
            "slot_of": slot_of}


def moe_route_scored_backward(logits: torch.Tensor, selected: torch.Tensor, dweights: torch.Tensor,
                              score: str = "softmax", renorm: bool = True,
                              scale: float = 1.0) -> torch.Tensor:
    """Gradient of moe_route_scored's logits [rows, E] (their dtype) from that of its weights
    (nsosx_moe_route_scored_backward); the balance bias has none."""
    fn = "moe_route_scored_backward"
    stride = _logit_rows(fn, logits)
    rows, e = logits.shape
    if selected.dim() != 2 or selected.shape[0] != rows or selected.shape[1] < 1:
        raise ValueError(f"{fn}: selected must be [rows, k], got {tuple(selected.shape)}")
    k = selected.shape[1]
    sig = _score_mode(fn, score)
    dev = logits.get_device()
    _on(fn, dev, ("selected", selected, torch.int32, None),
        ("dweights", dweights, torch.float32, (rows, k)))
    out = logits.new_empty((rows, e))
    call("nsosx_moe_route_scored_backward", _p(logits), _dt(logits), stride, _p(selected),
         _p(dweights), rows, e, k, sig, int(renorm), float(scale), _p(out), _stream_on(dev))
    return out


def _sequences(fn: str, cu_seqlens) -> int:
    """Sequences of a packed batch's bounds [S + 1]."""
    shape = () if cu_seqlens is None else cu_seqlens.shape
    if len(shape) != 1 or shape[0] < 1:
        raise ValueError(f"{fn}: cu_seqlens must be [sequences + 1], got {tuple(shape)}")
    if shape[0] >> 31:
        raise _too_many(fn, "cu_seqlens", shape)
    return shape[0] - 1


def _segments(fn: str, cu_seqlens, dev: int) -> int:
    """Sequences of a packed batch's bounds int32 [S + 1] (None: the batch is one)."""
    if cu_seqlens is None:
        return 1
    s = _sequences(fn, cu_seqlens)
    _on(fn, dev, ("cu_seqlens", cu_seqlens, torch.int32, None))
    return s


def moe_balance_loss(logits: torch.Tensor, selected: torch.Tensor, score: str = "softmax",
                     cu_seqlens=None, valid_rows=None) -> dict:
    """The router's balance loss E sum_e f_e P_e (nsosx_moe_balance_loss): f_e the share of the
    choices that fell on expert e, P_e its mean probability (softmax, or sigmoids over their sum);
    over the whole batch, or with cu_seqlens int32 [S + 1] per sequence and averaged over the
    sequences that have a valid row.

    logits f32 or bf16 [rows, E], selected int32 [rows, k] as moe_route_scored gives it.
    -> loss f32 [1], counts int32 [S, E], tokens int32 [S] (valid rows), mean_prob f32 [S, E], with
    S = 1 for the whole batch.  valid_rows as moe_route.  No autograd:
    moe_balance_loss_backward gives the logits' gradient."""
    fn = "moe_balance_loss"
    stride = _logit_rows(fn, logits)
    rows, e = logits.shape
    shape = selected.shape
    if len(shape) != 2 or shape[0] != rows or shape[1] < 1:
        raise ValueError(f"{fn}: selected must be [rows, k], got {tuple(shape)}")
    k = shape[1]
    sig = _score_mode(fn, score)
    dev = logits.get_device()
    mask = valid_rows_mask(valid_rows, rows, logits.device)
    _on(fn, dev, ("selected", selected, torch.int32, None), ("valid_rows", mask, torch.uint8, None))
    s = _segments(fn, cu_seqlens, dev)
    # (tensors of their own: a loss that is kept keeps nothing else, no workspace above all)
    loss = logits.new_empty(1, dtype=torch.float32)
    mean, counts, tokens = loss.new_empty((s, e)), selected.new_empty((s, e)), selected.new_empty(s)
    ws = selected.new_empty((lib().nsosx_moe_balance_loss_workspace(rows, e, s) + 3) // 4)
    call("nsosx_moe_balance_loss", _p(logits), _dt(logits), stride, _p(selected), _p(mask), rows, e, k,
         sig, _p(cu_seqlens), s, _p(loss), _p(counts), _p(tokens), _p(mean), _p(ws), _stream_on(dev))
    return {"loss": loss, "counts": counts, "tokens": tokens, "mean_prob": mean}


def moe_balance_loss_backward(logits: torch.Tensor, counts: torch.Tensor, tokens: torch.Tensor, k: int,
                              score: str = "softmax", cu_seqlens=None, valid_rows=None, dloss=1.0,
                              add=None) -> torch.Tensor:
    """Gradient of moe_balance_loss's logits [rows, E] (their dtype) times dloss, a number or a
    device f32 tensor of one element (nsosx_moe_balance_loss_backward); counts and tokens are the
    forward's, k its choices a row.  add: a gradient of the same shape and dtype
    (moe_route_scored_backward's) that is added to it."""
    fn = "moe_balance_loss_backward"
    stride = _logit_rows(fn, logits)
    rows, e = logits.shape
    sig = _score_mode(fn, score)
    dev = logits.get_device()
    mask = valid_rows_mask(valid_rows, rows, logits.device)
    s = _segments(fn, cu_seqlens, dev)
    scalar = dloss if isinstance(dloss, torch.Tensor) else None
    if scalar is not None and scalar.numel() != 1:
        raise ValueError(f"{fn}: dloss must hold one element, got {tuple(scalar.shape)}")
    _on(fn, dev, ("counts", counts, torch.int32, (s, e)), ("tokens", tokens, torch.int32, (s,)),
        ("valid_rows", mask, torch.uint8, None), ("dloss", scalar, torch.float32, None),
        ("add", add, logits.dtype, (rows, e)))
    out = logits.new_empty((rows, e))
    call("nsosx_moe_balance_loss_backward", _p(logits), _dt(logits), stride, _p(counts), _p(tokens),
         _p(mask), rows, e, k, sig, _p(cu_seqlens), s, 1.0 if scalar is not None else float(dloss),
         _p(scalar), _p(add), _p(out), _stream_on(dev))
    return out


def _combine_shapes(fn, expert_out, slot_of, weights):
    if expert_out.dim() != 2 or slot_of.dim() != 2 or 0 in expert_out.shape or 0 in slot_of.shape:
        raise ValueError(f"{fn}: expert_out must be [slots, dim] and slot_of [rows, k]")
    _on(fn, expert_out.get_device(), ("expert_out", expert_out, None, None),
        ("slot_of", slot_of, torch.int32, None), ("weights", weights, torch.float32, slot_of.shape))
    return (*slot_of.shape, *expert_out.shape)


def moe_combine_topk(expert_out: torch.Tensor, slot_of: torch.Tensor, weights: torch.Tensor,
                     out_dtype=torch.float32) -> torch.Tensor:
    """out[r] = sum_i weights[r, i] * expert_out[slot_of[r, i]] (nsosx_moe_combine_topk): the
    combine of moe_route_scored's weights [rows, k]; slot -1 adds nothing.  No autograd: the result
    is detached, moe_combine_topk_backward gives both gradients."""
    fn = "moe_combine_topk"
    rows, k, slots, dim = _combine_shapes(fn, expert_out, slot_of, weights)
    if out_dtype not in _DT:
        raise ValueError(f"{fn}: out_dtype must be float32 or bfloat16")
    out = expert_out.new_empty((rows, dim), dtype=out_dtype)
    call("nsosx_moe_combine_topk", _p(expert_out), _dt(expert_out), _p(slot_of), _p(weights), rows,
         slots, k, dim, _p(out), _DT[out_dtype], _stream_on(expert_out.get_device()))
    return out


def moe_combine_topk_backward(dout: torch.Tensor, expert_out: torch.Tensor, slot_of: torch.Tensor,
                              weights: torch.Tensor, perm=None) -> tuple:
    """Gradients of moe_combine_topk -> (dexpert_out [slots, dim] in expert_out's dtype, dweights
    f32 [rows, k]).  Rows of expert_out that no row holds get zeros: those with perm -1 where the
    routing's perm is given, else all are cleared first."""
    fn = "moe_combine_topk_backward"
    rows, k, slots, dim = _combine_shapes(fn, expert_out, slot_of, weights)
    dev = expert_out.get_device()
    _on(fn, dev, ("dout", dout, None, (rows, dim)), ("perm", perm, torch.int32, (slots,)))
    de = torch.empty_like(expert_out) if perm is not None else torch.zeros_like(expert_out)
    dw = weights.new_empty((rows, k))
    call("nsosx_moe_combine_topk_backward", _p(dout), _dt(dout), _p(expert_out), _dt(expert_out),
         _p(slot_of), _p(weights), _p(perm), rows, slots, k, dim, _p(de), _p(dw), _stream_on(dev))
    return de, dw


def int8_gemm(q: torch.Tensor, act_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
              bias=None, out_dtype=torch.float32) -> torch.Tensor:
    """y = (q @ w^T) * act_scale[:, None] * w_scale (+ bias) (nsosx_int8_gemm): int8 codes q
    [M, K] and weights w [N, K], a scale per token and per output, both as
    quantize_activations_bitnet gives them; y [M, N] f32 or bf16.  It has no gradient."""
    fn = "int8_gemm"
    if q.dim() != 2 or w.dim() != 2 or q.shape[1] != w.shape[1] or not (q.numel() and w.numel()):
        raise ValueError(f"{fn}: q [M, K] and w [N, K] must agree in K, got {tuple(q.shape)} and "
                         f"{tuple(w.shape)}")
    m, k = q.shape
    n = w.shape[0]
    dev = q.get_device()
    _on(fn, dev, ("q", q, torch.int8, None), ("act_scale", act_scale, torch.float32, (m,)),
        ("w", w, torch.int8, None), ("w_scale", w_scale, torch.float32, (n,)),
        ("bias", bias, torch.float32, (n,)))
    if out_dtype not in _DT:
        raise ValueError(f"{fn}: out_dtype must be float32 or bfloat16")
    y = q.new_empty((m, n), dtype=out_dtype)
    call("nsosx_int8_gemm", _p(q), _p(act_scale), _p(w), _p(w_scale), _p(bias), m, k, n, _p(y),
         _DT[out_dtype], _stream_on(dev))
    return y


def grouped_int8_gemm(q: torch.Tensor, act_scale: torch.Tensor, w: torch.Tensor,
                      w_scale: torch.Tensor, offsets: torch.Tensor, perm=None, bias=None,
                      squared_relu: bool = False, out_dtype=torch.float32) -> torch.Tensor:
    """int8_gemm of every expert's rows (nsosx_grouped_int8_gemm): w [E, N, K], w_scale and bias
    [E, N], the segments offsets [E+1] and, where q holds the unrouted rows, the slots' rows
    perm (else q is in slot order).  -> y [slots, N]; rows past offsets[E] are not written.  It has
    no gradient."""
    fn = "grouped_int8_gemm"
    if q.dim() != 2 or w.dim() != 3 or q.shape[1] != w.shape[2] or not (q.numel() and w.numel()):
        raise ValueError(f"{fn}: q [rows, K] and w [E, N, K] must agree in K, got "
                         f"{tuple(q.shape)} and {tuple(w.shape)}")
    rows, k = q.shape
    e, n, _ = w.shape
    slots = rows if perm is None else perm.numel()
    if slots == 0:
        raise ValueError(f"{fn}: perm must hold the slots' rows")
    dev = q.get_device()
    _on(fn, dev, ("q", q, torch.int8, None), ("act_scale", act_scale, torch.float32, (rows,)),
        ("w", w, torch.int8, None), ("w_scale", w_scale, torch.float32, (e, n)),
        ("offsets", offsets, torch.int32, (e + 1,)), ("perm", perm, torch.int32, (slots,)),
        ("bias", bias, torch.float32, (e, n)))
    if out_dtype not in _DT:
        raise ValueError(f"{fn}: out_dtype must be float32 or bfloat16")
    y = q.new_empty((slots, n), dtype=out_dtype)
    call("nsosx_grouped_int8_gemm", _p(q), _p(act_scale), rows, _p(w), _p(w_scale), _p(bias),
         _p(offsets), _p(perm), slots, e, k, n, int(squared_relu), _p(y), _DT[out_dtype],
         _stream_on(dev))
    return y


# ---- row norms of the hybrid block --------------------------------------------

def rmsnorm_gated(y: torch.Tensor, z=None, gamma=None, eps: float = 1e-5,
                  out_dtype=None) -> torch.Tensor:
    """RMSNorm(y * SiLU(z)) * gamma (src/mamba2.cpp:2677-2680); z None: rmsnorm(y) * gamma."""
    _dev(y, "y")
    if y.dim() != 2:
        raise ValueError("rmsnorm_gated: y must be [rows, dim]")
    if z is not None:
        _dev(z, "z", y.dtype)
        if z.shape != y.shape:
            raise ValueError("rmsnorm_gated: z must match y")
    _opt(gamma, "gamma")
    if gamma is not None and gamma.numel() != y.shape[1]:
        raise ValueError("rmsnorm_gated: gamma must have dim elements")
    out = torch.empty(y.shape, dtype=out_dtype or y.dtype, device=y.device)
    call("nsosx_rmsnorm_gated", _p(y), _p(z), _p(gamma), y.shape[0], y.shape[1], eps, _dt(y),
         _p(out), _dt(out), _stream())
    return out


def rmsnorm_gated_quant(y: torch.Tensor, z=None, gamma=None, eps: float = 1e-5, bits: int = 8,
                        want_out: bool = False, out_dtype=None):
    """rmsnorm_gated + the next BitLinear's int8 input quantization (src/mamba2.cpp:2677-2681,
    src/bitlinear.cpp:240-291) -> (q int8 [rows, dim], act_scale f32 [rows], normed or None).
    The normed rows are stored only with want_out (or where the one-pass form does not
    apply: dim % 512 != 0 or dim > 4096)."""
    _dev(y, "y")
    if y.dim() != 2:
        raise ValueError("rmsnorm_gated_quant: y must be [rows, dim]")
    if z is not None:
        _dev(z, "z", y.dtype)
        if z.shape != y.shape:
            raise ValueError("rmsnorm_gated_quant: z must match y")
    _opt(gamma, "gamma")
    rows, dim = y.shape
    if gamma is not None and gamma.numel() != dim:
        raise ValueError("rmsnorm_gated_quant: gamma must have dim elements")
    odt = out_dtype or y.dtype
    one_pass = dim % 512 == 0 and dim <= 4096
    out = torch.empty(y.shape, dtype=odt, device=y.device) if (want_out or not one_pass) else None
    q = torch.empty((rows, dim), dtype=torch.int8, device=y.device)
    s = torch.empty(rows, dtype=torch.float32, device=y.device)
    call("nsosx_rmsnorm_gated_quant", _p(y), _p(z), _p(gamma), rows, dim, eps, _dt(y), _p(out),
         _DT[odt], bits, _p(q), _p(s), _stream())
    return q, s, out


def add_rmsnorm(x: torch.Tensor, delta: torch.Tensor, gamma=None, eps: float = 1e-6,
                want_norm: bool = True):
    """residual = x + delta; norm = rmsnorm(residual) * gamma (src/jamba.cpp:3253, 3286-3290).

    Returns (residual, norm) with norm None when want_norm is False."""
    _dev(x, "x")
    _dev(delta, "delta", x.dtype)
    if x.dim() != 2 or delta.shape != x.shape:
        raise ValueError("add_rmsnorm: x and delta must be the same [rows, dim]")
    _opt(gamma, "gamma")
    res = torch.empty_like(x)
    norm = torch.empty_like(x) if want_norm else None
    call("nsosx_add_rmsnorm", _p(x), _p(delta), _p(gamma), x.shape[0], x.shape[1], eps, _dt(x),
         _p(res), _p(norm), _stream())
    return res, norm


# ---- layer norm and its gradients -------------------------------------------------

def _norm_rows(fn: str, x: torch.Tensor) -> tuple:
    """Rows, dim and type of x."""
    shape = x.shape
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError(f"{fn}: x must be [rows, dim], got {tuple(shape)}")
    rows, dim = shape
    if (rows | dim) >> 31:
        raise _too_many(fn, "x", shape)
    return rows, dim, _dt(x)


def layernorm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, out_dtype=None,
              want_stats: bool = False):
    """y = (x - mean) * rstd * weight + bias over the last dimension (nsosx_layernorm): x f32 or
    bf16 [rows, dim], weight and bias f32 [dim] or None.  -> y, or with want_stats (y, mean, rstd),
    f32 [rows] each, which layernorm_backward takes.  No autograd."""
    fn = "layernorm"
    rows, dim, dt = _norm_rows(fn, x)
    odt = out_dtype or x.dtype
    if odt not in _DT:
        raise ValueError(f"{fn}: out_dtype must be float32 or bfloat16")
    dev = x.get_device()
    _on(fn, dev, ("x", x, None, None), ("weight", weight, torch.float32, (dim,)),
        ("bias", bias, torch.float32, (dim,)))
    y = x.new_empty((rows, dim), dtype=odt)
    mean = rstd = None
    if want_stats:
        mean, rstd = x.new_empty((2, rows), dtype=torch.float32).unbind(0)
    call("nsosx_layernorm", _p(x), None, _p(weight), _p(bias), rows, dim, eps, dt, None, _p(y),
         _DT[odt], _p(mean), _p(rstd), _stream_on(dev))
    return (y, mean, rstd) if want_stats else y


def add_layernorm(x: torch.Tensor, delta: torch.Tensor, weight=None, bias=None, eps: float = 1e-5,
                  want_stats: bool = False) -> tuple:
    """residual = x + delta, y = layernorm(residual as stored), in one pass (nsosx_layernorm).
    -> (residual, y), or with want_stats (residual, y, mean, rstd)."""
    fn = "add_layernorm"
    rows, dim, dt = _norm_rows(fn, x)
    dev = x.get_device()
    _on(fn, dev, ("x", x, None, None), ("delta", delta, x.dtype, (rows, dim)),
        ("weight", weight, torch.float32, (dim,)), ("bias", bias, torch.float32, (dim,)))
    res, y = torch.empty_like(x), torch.empty_like(x)
    mean = rstd = None
    if want_stats:
        mean, rstd = x.new_empty((2, rows), dtype=torch.float32).unbind(0)
    call("nsosx_layernorm", _p(x), _p(delta), _p(weight), _p(bias), rows, dim, eps, dt, _p(res),
         _p(y), dt, _p(mean), _p(rstd), _stream_on(dev))
    return (res, y, mean, rstd) if want_stats else (res, y)


def layernorm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                       weight=None, dresidual=None, want_params: bool = True) -> dict:
    """Gradients of layernorm / add_layernorm (nsosx_layernorm_backward): x the normed rows (the
    residual, where there was an add), mean and rstd as the forward gave them.  -> dx (x's dtype;
    of both x and delta of an add) and, with want_params, dweight and dbias f32 [dim].  dresidual:
    the gradient that reached the residual by another way, added to dx."""
    fn = "layernorm_backward"
    rows, dim, dt = _norm_rows(fn, x)
    gdt = _dt(dy)
    dev = x.get_device()
    _on(fn, dev, ("x", x, None, None), ("dy", dy, None, (rows, dim)),
        ("mean", mean, torch.float32, (rows,)), ("rstd", rstd, torch.float32, (rows,)),
        ("weight", weight, torch.float32, (dim,)), ("dresidual", dresidual, x.dtype, (rows, dim)))
    dx = torch.empty_like(x)
    dw = db = ws = None
    if want_params:
        # (f32 tensors of their own: a gradient that is kept keeps no partial sums)
        dw, db = mean.new_empty(dim), mean.new_empty(dim)
        ws = mean.new_empty(lib().nsosx_layernorm_backward_workspace(rows, dim) // 4)
    call("nsosx_layernorm_backward", _p(dy), gdt, _p(x), _p(mean), _p(rstd), _p(weight),
         _p(dresidual), rows, dim, dt, _p(dx), _p(dw), _p(db), _p(ws), _stream_on(dev))
    return {"dx": dx, "dweight": dw, "dbias": db} if want_params else {"dx": dx}


# ---- gated linear recurrence --------------------------------------------------------

def _rec_view(fn: str, dev: int, name: str, t: torch.Tensor, dtype, shape) -> int:
    """Checks a [T, D] view with unit column stride (a column slice is fine); its row stride."""
    # (one line where all is well, as in _on)
    if t.get_device() == dev >= 0 and t.dtype == dtype and t.shape == shape:
        rs, cs = t.stride()
        if cs == 1 and rs >= shape[1]:
            return rs
    if t.get_device() != dev or dev < 0:
        raise ValueError(f"{fn}: {name} must be a device tensor on x's device")
    if t.dtype != dtype or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{fn}: {name} must be {tuple(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}")
    rows, d = shape
    # (a stride over one element says nothing)
    if (d > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < d):
        raise ValueError(f"{fn}: {name} needs unit column stride and rows that do not overlap")
    return t.stride(0) if rows > 1 else d


def _rec_inputs(fn: str, x, rg, ig, lam, *more) -> tuple:
    """Checks the recurrence's inputs and `more` as _on takes it; device, type and row strides."""
    shape = x.shape
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError(f"{fn}: x must be [tokens, dim], got {tuple(shape)}")
    if (shape[0] | shape[1]) >> 31:
        raise _too_many(fn, "x", shape)
    dt = _dt(x)
    if not x.is_cuda:
        raise ValueError("x must be a device tensor")
    dev = x.get_device()
    dtype = x.dtype
    xs, rs = _rec_view(fn, dev, "x", x, dtype, shape), _rec_view(fn, dev, "rg", rg, dtype, shape)
    igs = _rec_view(fn, dev, "ig", ig, dtype, shape)
    _on(fn, dev, ("lam", lam, torch.float32, shape[1:]), *more)
    return dev, dt, xs, rs, igs


def gated_recurrence(x: torch.Tensor, rg: torch.Tensor, ig: torch.Tensor, lam: torch.Tensor,
                     cu_seqlens: torch.Tensor, rate: float = 8.0, initial_state=None,
                     want_final: bool = True, want_carry: bool = False, out=None,
                     zero_rest=None) -> tuple:
    """Gated linear recurrence over a packed ragged batch (nsosx_gated_recurrence):

        a = exp(-rate softplus(lam) sigmoid(rg)),  h_t = a_t h_(t-1) + sqrt(1 - a_t^2) sigmoid(ig_t) x_t

    x, the decay gate's logits rg and the input gate's ig f32 or bf16 [T, D] (column slices are
    fine), lam f32 [D], cu_seqlens int32 [S + 1], initial_state f32 [S, D] or None.  -> (y [T, D] in
    x's dtype, final_state f32 [S, D] or None), and with want_carry a third tensor that
    gated_recurrence_backward takes.  out: a [T, D] view to write y into.  zero_rest: rows of no
    sequence become zeros (a fresh y's by default) or stay as they were (out's).  No autograd."""
    fn = "gated_recurrence"
    s = _sequences(fn, cu_seqlens)
    dev, dt, xs, rs, igs = _rec_inputs(fn, x, rg, ig, lam, ("cu_seqlens", cu_seqlens, torch.int32, None),
                                       ("initial_state", initial_state, torch.float32, (s, *x.shape[1:])))
    t, d = x.shape
    y = x.new_empty((t, d)) if out is None else out
    ys = d if out is None else _rec_view(fn, dev, "out", out, x.dtype, (t, d))
    final = x.new_empty((s, d), dtype=torch.float32) if want_final else None
    tiles = -(-t // lib().nsosx_gated_recurrence_tile())
    carry = x.new_empty((tiles, d), dtype=torch.float32) if want_carry else None
    ws = x.new_empty(int(lib().nsosx_gated_recurrence_workspace(t, d)), dtype=torch.uint8)
    call("nsosx_gated_recurrence", _p(x), xs, _p(rg), rs, _p(ig), igs, _p(lam), rate, _p(cu_seqlens), s,
         t, d, dt, _p(initial_state), int(out is None if zero_rest is None else zero_rest), _p(y), ys,
         _p(final), _p(carry), _p(ws), _stream_on(dev))
    return (y, final, carry) if want_carry else (y, final)


def gated_recurrence_backward(dy: torch.Tensor, x: torch.Tensor, rg: torch.Tensor, ig: torch.Tensor,
                              lam: torch.Tensor, cu_seqlens: torch.Tensor, carry: torch.Tensor,
                              rate: float = 8.0, initial_state=None, dfinal=None, out=None,
                              zero_rest=None) -> dict:
    """Gradients of gated_recurrence (nsosx_gated_recurrence_backward) from dy [T, D] (x's dtype) and,
    where the final states went on, dfinal f32 [S, D]; carry is the forward's, the rest its
    arguments.  -> dx, drg, dig [T, D], dlam f32 [D] and, with an initial_state or dfinal, dinitial f32
    [S, D].  out: three [T, D] views (dx, drg, dig) to write into, side by side in one buffer for
    one.  zero_rest as in gated_recurrence."""
    fn = "gated_recurrence_backward"
    s, f32 = _sequences(fn, cu_seqlens), torch.float32
    t, d = x.shape if x.dim() == 2 else (0, 0)
    tiles = -(-t // lib().nsosx_gated_recurrence_tile())
    dev, dt, xs, rs, igs = _rec_inputs(fn, x, rg, ig, lam, ("cu_seqlens", cu_seqlens, torch.int32, None),
                                       ("carry", carry, f32, (tiles, d)),
                                       ("initial_state", initial_state, f32, (s, d)), ("dfinal", dfinal, f32, (s, d)))
    dys = _rec_view(fn, dev, "dy", dy, x.dtype, x.shape)
    if out is None:
        grads, gs = x.new_empty((3, t, d)).unbind(0), (d, d, d)
    else:
        if len(out) != 3:
            raise ValueError(f"{fn}: out must hold dx, drg and dig")
        grads = out
        gs = [_rec_view(fn, dev, "out", g, x.dtype, (t, d)) for g in out]
    dlam = lam.new_empty(d)
    want0 = initial_state is not None or dfinal is not None
    dinit = lam.new_empty((s, d)) if want0 else None
    ws = x.new_empty(int(lib().nsosx_gated_recurrence_backward_workspace(t, d)), dtype=torch.uint8)
    call("nsosx_gated_recurrence_backward", _p(dy), dys, _p(x), xs, _p(rg), rs, _p(ig), igs, _p(lam),
         rate, _p(cu_seqlens), s, t, d, dt, _p(initial_state), _p(carry), _p(dfinal),
         int(out is None if zero_rest is None else zero_rest),
         _p(grads[0]), gs[0], _p(grads[1]), gs[1], _p(grads[2]), gs[2], _p(dlam), _p(dinit), _p(ws),
         _stream_on(dev))
    r = {"dx": grads[0], "drg": grads[1], "dig": grads[2], "dlam": dlam}
    if want0:
        r["dinitial"] = dinit
    return r


def gated_recurrence_step(x: torch.Tensor, rg: torch.Tensor, ig: torch.Tensor, lam: torch.Tensor,
                          state: torch.Tensor, rate: float = 8.0, state_out=None) -> torch.Tensor:
    """One token per row through gated_recurrence (nsosx_gated_recurrence_step): x, rg, ig [R, D],
    state f32 [R, D], updated in place or written to state_out.  -> y [R, D] in x's dtype."""
    fn = "gated_recurrence_step"
    f32 = torch.float32
    dev, dt, xs, rs, igs = _rec_inputs(fn, x, rg, ig, lam, ("state", state, f32, x.shape),
                                       ("state_out", state_out, f32, x.shape))
    r, d = x.shape
    if state_out is None:
        state_out = state
    y = x.new_empty((r, d))
    call("nsosx_gated_recurrence_step", _p(x), xs, _p(rg), rs, _p(ig), igs, _p(lam), rate, r, d, dt,
         _p(state), _p(state_out), _p(y), d, _stream_on(dev))
    return y


# ---- the decode conv ring -----------------------------------------------------

def conv_step(x: torch.Tensor, weight: torch.Tensor, bias, ring, apply_silu: bool = True,
              out_dtype=None) -> torch.Tensor:
    """Decode conv ring step in place on `ring` [R, W-1, C] (src/mamba2.cpp:4072-4090) -> out."""
    if not x.is_cuda or x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("conv_step: x must be a device [rows, channels] with unit channel stride")
    _dev(weight, "weight", torch.float32)
    _opt(bias, "bias")
    r, c = x.shape
    w = weight.shape[1]
    if weight.shape[0] != c:
        raise ValueError("conv_step: weight must be [channels, W]")
    if w > 1:
        _dev(ring, "ring", torch.float32)
        if tuple(ring.shape) != (r, w - 1, c):
            raise ValueError("conv_step: ring must be [rows, W-1, channels]")
    out = torch.empty((r, c), dtype=out_dtype or x.dtype, device=x.device)
    call("nsosx_conv_step", _p(x), _dt(x), x.stride(0), r, c, _p(weight), _p(bias), w,
         _p(ring) if w > 1 else None, int(apply_silu), _p(out), _dt(out), _stream())
    return out


# ---- quantization-aware training (fake quant + STE clip) -------------------------

def qat_fake_quant_ternary(w: torch.Tensor, scale: float) -> torch.Tensor:
    """qat_fake_quant_ternary (src/bitnet_gpu_dispatch.cpp:193-217): ternary(w / scale) * scale."""
    _dev(w, "w", torch.float32)
    out = torch.empty_like(w)
    call("nsosx_qat_fake_quant_ternary", _p(w), w.numel(), float(scale), _p(out), _stream())
    return out


def qat_fake_quant_ternary_absmean(w: torch.Tensor):
    """qat_fake_quant_ternary_absmean (src/bitnet_gpu_dispatch.cpp:219-245) -> (out, scale [1])
    with the absmean scale computed and kept on the device."""
    _dev(w, "w", torch.float32)
    out = torch.empty_like(w)
    scale = torch.empty(1, dtype=torch.float32, device=w.device)
    ws = torch.empty(int(lib().nsosx_qat_absmean_workspace(w.numel())), dtype=torch.uint8,
                     device=w.device)
    call("nsosx_qat_fake_quant_ternary_absmean", _p(w), w.numel(), _p(out), _p(scale), _p(ws),
         _stream())
    return out, scale


def qat_fake_quant_activations(x: torch.Tensor, precision_bits: int = 8) -> torch.Tensor:
    """qat_fake_quant_activations (src/bitnet_gpu_dispatch.cpp:247-282): per-row absmax
    quantize-dequantize of the last dimension."""
    _dev(x, "x", torch.float32)
    k = x.shape[-1] if x.dim() else 0
    m = x.numel() // k if k else 0
    out = torch.empty_like(x)
    call("nsosx_qat_fake_quant_activations", _p(x), m, k, int(precision_bits), _p(out), _stream())
    return out


def qat_ste_clip_weight_grad(dW: torch.Tensor, w: torch.Tensor, scale) -> torch.Tensor:
    """qat_ste_clip_weight_grad(_device_scale) (src/bitnet_gpu_dispatch.cpp:284-325), in place
    on dW; `scale` is a float or a device tensor [1]."""
    _dev(dW, "dW", torch.float32)
    _dev(w, "w", torch.float32)
    if dW.shape != w.shape:
        raise ValueError("qat_ste_clip_weight_grad requires identical shapes")
    if isinstance(scale, torch.Tensor):
        _dev(scale, "scale", torch.float32)
        call("nsosx_qat_ste_clip_weight_grad", _p(dW), _p(w), w.numel(), 0.0, _p(scale), _stream())
    else:
        call("nsosx_qat_ste_clip_weight_grad", _p(dW), _p(w), w.numel(), float(scale), None,
             _stream())
    return dW
