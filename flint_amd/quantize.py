"""Host side of the int4 weight path: quantise / dequantise / M=1 and M=k GEMV, all on the GPU
through the C ABI, plus a drop-in for gpt-fast's WeightOnlyInt4Linear. Beside it 8-bit integers for
weights and activations both (DynamicInt8Linear): one scale per output channel and per token.

Mirrors reference engine/quantize.py:359-525 (prepare_int4_weight_and_scales_and_zeros,
linear_forward_int4, WeightOnlyInt4Linear): same groupsize (128), same quantised values,
same dequantised bf16 values; the packed layout is this library's own (see include/flint_amd.h).
"""
import os

import torch

from . import _lib

GROUP = _lib.GROUP

# the whole forward of WeightOnlyInt4Linear as one call of the torch extension, over the library
# beside it (not over another one that FLINT_AMD_LIB names)
_linear_fast = _int8_fast = None
if "FLINT_AMD_LIB" not in os.environ:
    try:
        from ._torch_ops import linear_fast as _linear_fast
        from ._torch_ops import int8_fast as _int8_fast
    except ImportError:
        pass


def _check_dev(t, dtype, name):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA (HIP) tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def quantize_int4(w, q=None, sz=None):
    """Quantise a bf16 [N, K] device matrix group-wise (128) to (q int32 [N, K/8], sz int32 [N, K/128])."""
    _check_dev(w, torch.bfloat16, "w")
    n, k = w.shape
    if k % GROUP:
        raise ValueError("K must be a multiple of 128")
    if q is None:
        q = torch.empty(n, k // 8, dtype=torch.int32, device=w.device)
    if sz is None:
        sz = torch.empty(n, k // GROUP, dtype=torch.int32, device=w.device)
    _lib.call("fl_quantize_int4", _lib.ptr(w), _lib.ptr(q), _lib.ptr(sz), n, k, _lib.stream_ptr())
    return q, sz


def dequantize_int4(q, sz, matrix_cores=False):
    """Bit-exact bf16 [N, K] dequantisation through the kernels' own device routine: the vector-ALU
    form (fl_gemm_int4's) or, with matrix_cores, the lane-by-lane MFMA form of the decode GEMVs and
    fl_gemv_int4."""
    _check_dev(q, torch.int32, "q")
    _check_dev(sz, torch.int32, "sz")
    n, k = q.shape[0], q.shape[1] * 8
    out = torch.empty(n, k, dtype=torch.bfloat16, device=q.device)
    _lib.call("fl_dequant_int4_mx" if matrix_cores else "fl_dequant_int4", _lib.ptr(q), _lib.ptr(sz),
              _lib.ptr(out), n, k, _lib.stream_ptr())
    return out


def tile_int4(q, qt=None):
    """The tiled layout (fl_tile_int4) of a row-layout int4 matrix q [..., N, K/8] (N % 16 == 0;
    leading dims are stacked rows): same shape and dtype, 1 KB per 16 rows x 128-group unit."""
    _check_dev(q, torch.int32, "q")
    k = q.shape[-1] * 8
    n = q.numel() // q.shape[-1]
    if n % 16:
        raise ValueError("tile_int4: the stacked row count must be a multiple of 16")
    if qt is None:
        qt = torch.empty_like(q)
    elif qt.shape != q.shape or qt.dtype != torch.int32 or not qt.is_contiguous():
        raise ValueError("tile_int4: qt must be a contiguous int32 tensor shaped like q")
    _lib.call("fl_tile_int4", _lib.ptr(q), _lib.ptr(qt), n, k, _lib.stream_ptr())
    return qt


def gemv_int4(q, sz, x, y=None):
    """y[N] = bf16(x[K] . dq[N,K]^T) with fp32 accumulation (M = 1)."""
    _check_dev(q, torch.int32, "q")
    _check_dev(sz, torch.int32, "sz")
    _check_dev(x, torch.bfloat16, "x")
    n, k = q.shape[0], q.shape[1] * 8
    if x.numel() != k:
        raise ValueError(f"x has {x.numel()} elements, expected {k}")
    if y is None:
        y = torch.empty(n, dtype=torch.bfloat16, device=q.device)
    _lib.call("fl_gemv_int4", _lib.ptr(q), _lib.ptr(sz), _lib.ptr(x), _lib.ptr(y), n, k,
              _lib.stream_ptr())
    return y


def gemm_int4(q, sz, x, y=None):
    """Y[M,N] = bf16(X[M,K] . dq[N,K]^T) for any M: one fl_gemm_int4 launch up to 32 rows
    (FL_MAX_VERIFY), which reads the weights once for all of them; beyond, fl_gemm_rows_int4, which
    reads and dequantises them once per 64 or 128 rows (launches of 32 rows where it does not take the
    size or there is no memory for its workspace)."""
    _check_dev(q, torch.int32, "q")
    _check_dev(sz, torch.int32, "sz")
    _check_dev(x, torch.bfloat16, "x")
    n, k = q.shape[0], q.shape[1] * 8
    m = x.shape[0]
    if x.shape[1] != k:
        raise ValueError("x inner dimension mismatch")
    if y is None:
        y = torch.empty(m, n, dtype=torch.bfloat16, device=q.device)
    if m > 0 and (y.shape != (m, n) or not y.is_contiguous()):
        raise ValueError("y must be a contiguous [M, N] tensor")
    if m > _lib.MAX_VERIFY:
        need = _lib.ctypes.c_int64()
        if _lib.load().fl_gemm_rows_workspace(m, n, k, _lib.ctypes.byref(need)) == _lib.FL_OK:
            try:
                ws = torch.empty(need.value // 4, dtype=torch.float32, device=q.device) if need.value else None
            except torch.OutOfMemoryError:
                pass  # no room for the part sums: launches of 32 rows need none
            else:
                _lib.call("fl_gemm_rows_int4", _lib.ptr(q), _lib.ptr(sz), _lib.ptr(x), _lib.ptr(y), _lib.ptr(ws),
                          m, n, k, _lib.stream_ptr())
                return y
    for r0 in range(0, m, _lib.MAX_VERIFY):
        mb = min(_lib.MAX_VERIFY, m - r0)
        _lib.call("fl_gemm_int4", _lib.ptr(q), _lib.ptr(sz), _lib.ptr(x[r0:]), _lib.ptr(y[r0:]), mb, n, k,
                  _lib.stream_ptr())
    return y


# bit position of element e (0..7) inside its packed word: element 2i at 4i, 2i+1 at 16+4i
NIBBLE_SHIFT = [0, 16, 4, 20, 8, 24, 12, 28]


def unpack_q(q):
    """int32 [N, K/8] packed words -> int32 [N, K] values in [0, 15] (host-side inspection)."""
    shifts = torch.tensor(NIBBLE_SHIFT, device=q.device, dtype=torch.int32)
    v = (q.unsqueeze(-1) >> shifts) & 0xF
    return v.reshape(q.shape[0], q.shape[1] * 8)


def pack_q(vals):
    """int32 [N, K] values in [0, 15] -> int32 [N, K/8] packed words (inverse of unpack_q)."""
    n, k = vals.shape
    v = vals.to(torch.int64).view(n, k // 8, 8)
    shifts = torch.tensor(NIBBLE_SHIFT, device=vals.device, dtype=torch.int64)
    words = (v << shifts).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def unpack_sz(sz):
    """int32 [N, K/128] -> (scales bf16 [N, K/128], zeros bf16 [N, K/128])."""
    s = (sz & 0xFFFF).to(torch.int16).view(torch.bfloat16)
    z = ((sz >> 16) & 0xFFFF).to(torch.int16).view(torch.bfloat16)
    return s, z


def scales_and_zeros_gptfast(sz):
    """Our [N, K/128] scale/zero words -> gpt-fast's packed [K/128, N, 2] bf16 layout
    (reference engine/quantize.py:79-93 pack_scales_and_zeros)."""
    s, z = unpack_sz(sz)
    return torch.stack([s, z], dim=-1).transpose(0, 1).contiguous()


class WeightOnlyInt4Linear(torch.nn.Module):
    """Drop-in for reference engine/quantize.py:483-525 (groupsize 128), on the HIP GEMVs.

    forward(x [..., K] bf16) -> [..., N] bf16 for any M = prod(leading dims): the GEMV at M = 1, one
    weight read for up to 32 rows (speculative verify), the tiled GEMM for more (a prompt).
    """

    def __init__(self, in_features, out_features, bias=False, device=None, groupsize=GROUP):
        super().__init__()
        if bias:
            raise ValueError("require bias=False")
        if groupsize != GROUP:
            raise ValueError("groupsize must be 128")
        if in_features % GROUP:
            raise ValueError("in_features must be a multiple of 128")
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("weight", torch.zeros(out_features, in_features // 8,
                                                   dtype=torch.int32, device=device))
        self.register_buffer("scales_and_zeros", torch.zeros(out_features, in_features // GROUP,
                                                             dtype=torch.int32, device=device))

    @classmethod
    def from_float(cls, w):
        m = cls(w.shape[1], w.shape[0], device=w.device)
        quantize_int4(w.to(torch.bfloat16).contiguous(), m.weight, m.scales_and_zeros)
        return m

    def forward(self, x):
        if _linear_fast is not None and type(x) is torch.Tensor and x.is_cuda:
            y = _linear_fast(x, self.weight, self.scales_and_zeros,
                             torch._C._cuda_getCurrentRawStream(torch.cuda.current_device()))
            if y is not None:
                return y
        shape = x.shape
        x2 = x.reshape(-1, shape[-1]).to(torch.bfloat16).contiguous()
        if x2.shape[0] == 1:
            y = gemv_int4(self.weight, self.scales_and_zeros, x2.view(-1)).view(1, -1)
        else:
            y = gemm_int4(self.weight, self.scales_and_zeros, x2)
        return y.view(*shape[:-1], self.out_features)


# ---- 8-bit integers ------------------------------------------------------------------------------

def _check_int8(k):
    if k % 16 or not 16 <= k <= 65536:
        raise ValueError("K must be a multiple of 16, at most 65536")


def _check_weight(wq, ws):
    _check_dev(wq, torch.int8, "weight")
    _check_dev(ws, torch.float32, "scales")
    if wq.dim() != 2 or ws.shape != wq.shape[:1]:
        raise ValueError("weight must be [N, K] and scales [N]")
    _check_int8(wq.shape[1])
    if ws.device != wq.device:
        raise ValueError("weight and scales must be on one device")


def aligned16(t):
    """t, or a copy of it where its data does not start on 16 bytes (a view into a tensor may not). To be held in a
    name until the launch: a copy freed before it may be given to the next one, or to another thread."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def workspace(name, *sizes, device):
    """Device bytes for a call, of what the C entry `name` asks for (None where that is 0)."""
    need = _lib.ctypes.c_int64()
    _lib.call(name, *sizes, _lib.ctypes.byref(need))
    return torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None


def quantize_int8(x, q=None, scale=None):
    """Rows of a bf16 [M, K] device matrix in 8 bits: (q int8 [M, K], scale fp32 [M]), scale = max|row| times
    fp32(1 / 127) and q = row / scale rounded to the nearest, ties to even (fl_quantize_int8). (max|row| / 127 by a
    division is an ulp more for six of the 128 bf16 significands, and gives 63 for half of their maximum in place of 64.)
    For a weight matrix the rows are its output channels, for activations the tokens."""
    _check_dev(x, torch.bfloat16, "x")
    if x.dim() != 2:
        raise ValueError("x must be [M, K]")
    m, k = x.shape
    _check_int8(k)
    if q is None:
        q = torch.empty(m, k, dtype=torch.int8, device=x.device)
    if scale is None:
        scale = torch.empty(m, dtype=torch.float32, device=x.device)
    _check_dev(q, torch.int8, "q")
    _check_dev(scale, torch.float32, "scale")
    if q.shape != x.shape or scale.shape != x.shape[:1] or q.device != x.device or scale.device != x.device:
        raise ValueError("q must be [M, K] and scale [M], on x's device")
    if m:
        xa = aligned16(x)
        with torch.cuda.device(x.device):
            _lib.call("fl_quantize_int8", _lib.ptr(xa), _lib.ptr(q), _lib.ptr(scale), m, k, _lib.stream_ptr())
    return q, scale


def _check_out_dtype(out_dtype):
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("out_dtype must be torch.bfloat16 or torch.float32")


def gemm_int8(xq, xs, wq, ws, out_dtype=torch.bfloat16):
    """Y[M, N] = (xq . wq^T) * xs[:, None] * ws for 8-bit rows xq [M, K] and weights wq [N, K] with one fp32 scale
    per row (quantize_int8's). The integer sums are exact, so a row's result does not depend on the batch
    it is in. out_dtype: bf16, or fp32 (logits)."""
    f32 = out_dtype is torch.float32
    if _int8_fast is not None and xs is not None and xq.is_cuda and (f32 or out_dtype is torch.bfloat16):
        y = _int8_fast(xq, xs, wq, ws, f32, torch._C._cuda_getCurrentRawStream(xq.get_device()))
        if y is not None:
            return y
    _check_out_dtype(out_dtype)
    _check_weight(wq, ws)
    _check_dev(xq, torch.int8, "xq")
    _check_dev(xs, torch.float32, "xs")
    n, k = wq.shape
    if xq.dim() != 2 or xq.shape[1] != k or xs.shape != xq.shape[:1]:
        raise ValueError("xq must be [M, K] and xs [M]")
    if xq.device != wq.device or xs.device != wq.device:
        raise ValueError("xq, xs and weight must be on one device")
    m = xq.shape[0]
    y = torch.empty(m, n, dtype=out_dtype, device=xq.device)
    if m and n:
        xa, wa = aligned16(xq), aligned16(wq)
        with torch.cuda.device(xq.device):
            work = workspace("fl_gemm_int8_workspace", m, n, k, device=xq.device)
            _lib.call("fl_gemm_int8", _lib.ptr(xa), _lib.ptr(xs), _lib.ptr(wa), _lib.ptr(ws), _lib.ptr(y), int(f32),
                      _lib.ptr(work), m, n, k, _lib.stream_ptr())
    return y


def linear_int8(x, wq, ws, out_dtype=torch.bfloat16):
    """x [..., K] bf16 -> [..., N]: quantize_int8 of x's rows (tokens) and gemm_int8 with the weights, in one call
    (fl_linear_int8)."""
    f32 = out_dtype is torch.float32
    if _int8_fast is not None and x.is_cuda and (f32 or out_dtype is torch.bfloat16):
        y = _int8_fast(x, None, wq, ws, f32, torch._C._cuda_getCurrentRawStream(x.get_device()))
        if y is not None:
            return y
    _check_out_dtype(out_dtype)
    _check_weight(wq, ws)
    n, k = wq.shape
    if not x.is_cuda or x.dtype != torch.bfloat16:
        raise ValueError("x must be a torch.bfloat16 CUDA (HIP) tensor")
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x's last dimension must be {k}")
    if x.device != wq.device:
        raise ValueError("x and weight must be on one device")
    x2 = aligned16(x.detach().reshape(-1, k).contiguous())
    m = x2.shape[0]
    y = torch.empty(m, n, dtype=out_dtype, device=x.device)
    if m and n:
        wa = aligned16(wq)
        with torch.cuda.device(x.device):
            work = workspace("fl_linear_int8_workspace", m, n, k, device=x.device)
            _lib.call("fl_linear_int8", _lib.ptr(x2), _lib.ptr(wa), _lib.ptr(ws), _lib.ptr(y), int(f32),
                      _lib.ptr(work), m, n, k, _lib.stream_ptr())
    return y.view(*x.shape[:-1], n)


class DynamicInt8Linear(torch.nn.Module):
    """A linear with 8-bit integer weights (one scale per output channel) whose input rows are quantised on the
    way, one scale per token: the product runs on the integer matrix cores. For inference. The scales stay fp32 when a
    model that holds it is cast to another type.

    forward(x [..., K] bf16) -> [..., N] bf16, K a multiple of 16. For a vocabulary head whose logits are wanted in
    fp32 or as log probabilities: linear_int8(..., out_dtype=torch.float32), generate.head_logprobs.
    """

    def __init__(self, in_features, out_features, bias=False, device=None):
        super().__init__()
        if bias:
            raise ValueError("require bias=False")
        _check_int8(in_features)
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("weight", torch.zeros(out_features, in_features, dtype=torch.int8, device=device))
        self.register_buffer("scales", torch.zeros(out_features, dtype=torch.float32, device=device))

    def _apply(self, fn, recurse=True):
        scales = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype != torch.float32:  # the whole model was cast (to(bfloat16), half()): the scales are not
            self.scales = scales.to(self.scales.device)
        return self

    @classmethod
    def from_float(cls, w):
        m = cls(w.shape[1], w.shape[0], device=w.device)
        quantize_int8(w.detach().to(torch.bfloat16).contiguous(), m.weight, m.scales)
        return m

    def forward(self, x):
        return linear_int8(x.to(torch.bfloat16), self.weight, self.scales)
