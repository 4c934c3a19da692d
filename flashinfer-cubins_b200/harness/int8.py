"""Products of 8-bit integers with a scale for each token and each output channel, the quantiser
in front of them, and the norms around a block: the serving path of models whose weights are
INT8, beside the NVFP4 one of this package.

    codes, scales = int8.quantize_tokens(x)                       # a row's scale: max |x| / 127
    h = int8.gemm(codes, w13, scales, w13_scales, gated=True)     # silu(gate) * up in the epilogue
    y = int8.grouped_gemm(rows, w, rows_scales, w_scales, offsets)  # ragged rows per expert
    r, n, s = int8.residual_norm(y, residual, post_weight=..., next_weight=..., quantize=True)

Each call is one launch, asynchronous on the current stream of its tensors' device (made current
for the launch where it is not), without a workspace, a plan or anything kept for the next call: it
can be captured in a CUDA graph and called from several threads and streams at once. A call with
wrong operands raises ``ValueError`` before anything is launched, one on a device that is not
compute capability 10.0 ``RuntimeError``. There are no derivatives: operands that require a gradient
are refused while gradients are recorded, operands with a tangent of forward differentiation always.

Codes are ``torch.int8`` ``[rows, k]`` whose rows start 16-byte aligned and a multiple of 16 bytes
apart, which is what ``quantize_tokens`` and ``residual_norm`` return for every ``k`` (a view of
padded rows where ``k`` is no multiple of 16; ``empty_codes`` makes such a buffer). Scales are FP32
and contiguous. Weights are quantised by the same function, a scale for each output channel:
``quantize_tokens(w)``.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import native

OUT_KINDS = {torch.float16: native.OUT_F16, torch.float32: native.OUT_F32,
             torch.bfloat16: native.OUT_BF16}
IN_KINDS = {torch.float32: native.IN_F32, torch.bfloat16: native.IN_BF16,
            torch.float16: native.IN_F16}
MAX_DEPTH = 131071  # k: sums of products of codes stay within 32 bits
MAX_EXPERTS = 1024
MAX_HIDDEN = 32768
MAX_ROWS = 1 << 30  # rows of an operand; n at most half of that

# Decode calls take a few microseconds on the GPU, so the host's share counts: devices are compared by
# index, the current stream's handle is read without making a Stream object (2 us), and a tensor's
# checks are one function call.
_INT8, _FLOAT = torch.int8, torch.float32
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_supported: dict[int, bool] = {}


def _check_device(index: int) -> None:
    if index < 0:
        raise RuntimeError("sm_100a code cannot run on the CPU")
    if index not in _supported:
        _supported[index] = native.device_supported(index)
    if not _supported[index]:
        raise RuntimeError(f"sm_100a code cannot run on cuda:{index}")


def _launch(index: int, entry: str, *arguments) -> None:
    """Call a C entry point on device ``index`` and its current stream."""
    function = getattr(native.load(), entry)
    if index == _current_device():
        status = function(*arguments, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = function(*arguments, _raw_stream(index))
    if status:
        native.check(status)


def _refuse_gradients() -> None:
    raise ValueError("the INT8 operators have no backward; call them under torch.no_grad()")


def refuse_tangents(*tensors: torch.Tensor | None) -> None:
    """Refuse operands of forward differentiation (which no_grad does not switch off)."""
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("the INT8 operators have no derivatives: an operand has a tangent")


def check_status(device: torch.device | str | int | None = None) -> None:
    """Synchronise ``device``'s current stream and raise ``native.NativeError`` if a product on it
    abandoned a bounded wait since the last call (its result is then undefined)."""
    with torch.cuda.device(device):
        value = native.ctypes.c_int(0)
        native.check(native.load().nvfp4_int8_status(_raw_stream(torch.cuda.current_device()),
                                                     native.ctypes.byref(value)))


def _too_many(what: str, count: int) -> None:
    raise ValueError(f"{what}: {count} rows, at most {MAX_ROWS}")


def _rows(t: torch.Tensor, shape, what: str) -> int:
    """Elements between the rows of ``t`` (its last but one dimension; ``shape`` is its shape)."""
    stride = t.stride()
    if stride[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{what}: elements of a row must be neighbours")
    return stride[-2] if shape[-2] > 1 else -(-shape[-1] // 16) * 16  # one row: nothing lies between


def _vector(t: torch.Tensor, shape: tuple, what: str, index: int) -> int:
    if t.dtype is not _FLOAT or t.shape != shape or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"{what}: expected contiguous float32 {shape} beside the first operand, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def empty_codes(rows: int, k: int, device: torch.device | str) -> torch.Tensor:
    """An INT8 ``[rows, k]`` buffer whose rows lie 16-byte aligned."""
    pitch = -(-k // 16) * 16
    if pitch == k:
        return torch.empty(rows, k, dtype=torch.int8, device=device)
    return torch.empty(rows, pitch, dtype=torch.int8, device=device)[:, :k]


def _codes(t: torch.Tensor, dims: int, what: str, index: int) -> int:
    shape = t.shape
    if t.dtype is not _INT8 or len(shape) != dims or t.get_device() != index:
        raise ValueError(f"{what}: expected {dims}-d int8 beside the first operand, got {t.dtype} "
                         f"{tuple(shape)} on {t.device}")
    stride = t.stride()
    if stride[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{what}: elements of a row must be neighbours")
    return stride[-2] if shape[-2] > 1 else -(-shape[-1] // 16) * 16


def _given(out: torch.Tensor, shape: tuple, dtype: torch.dtype, index: int, what: str) -> int:
    """Elements between the rows of an output that the caller gave."""
    if out.dtype is not dtype or out.shape != shape or out.get_device() != index:
        raise ValueError(f"{what}: expected {dtype} {shape} beside the first operand, got {out.dtype} "
                         f"{tuple(out.shape)} on {out.device}")
    return _rows(out, shape, what)


def _width(width: int, gated: bool) -> int:
    if gated and width % 2:
        raise ValueError(f"gated weights hold gate rows and as many up rows, got {width}")
    return width // 2 if gated else width


def gemm(a: torch.Tensor, b: torch.Tensor, a_scales: torch.Tensor, b_scales: torch.Tensor, *,
         bias: torch.Tensor | None = None, gated: bool = False,
         out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """``(a @ b.T) * a_scales[:, None] * b_scales + bias`` of INT8 codes ``a [m, k]`` and
    ``b [n, k]``, summed exactly in 32-bit integers and rounded once to ``out_dtype`` (FP16, BF16 or
    FP32). With ``gated`` ``b`` is ``[2n, k]``, gate rows before up rows, and the result
    ``silu(gate) * up`` ``[m, n]``. ``k`` and ``n`` are at least 1. ``out``: a tensor to write it to."""
    index = a.get_device()
    if torch.is_grad_enabled() and (a_scales.requires_grad or b_scales.requires_grad
                                    or (bias is not None and bias.requires_grad)
                                    or (out is not None and out.requires_grad)):
        _refuse_gradients()
    refuse_tangents(a_scales, b_scales, bias, out)
    lda, ldb = _codes(a, 2, "a", index), _codes(b, 2, "b", index)
    (m, k), (width, depth) = a.shape, b.shape
    if depth != k:
        raise ValueError(f"a is {k} deep, b {depth}")
    if m > MAX_ROWS or width > MAX_ROWS:
        _too_many("a or b", max(m, width))
    kind = OUT_KINDS.get(out_dtype)
    if kind is None:
        raise ValueError(f"no output in {out_dtype}")
    n = _width(width, gated)
    pa, pb = _vector(a_scales, (m,), "a_scales", index), _vector(b_scales, (width,), "b_scales", index)
    pbias = None if bias is None else _vector(bias, (width,), "bias", index)
    _check_device(index)
    if out is None:
        out, ldd = torch.empty(m, n, dtype=out_dtype, device=a.device), n
    else:
        ldd = _given(out, (m, n), out_dtype, index, "out")
    _launch(index, "nvfp4_int8_gemm", a.data_ptr(), lda, b.data_ptr(), ldb, pa, pb, pbias,
            out.data_ptr(), ldd, m, n, k, kind, gated)
    return out


def grouped_gemm(a: torch.Tensor, b: torch.Tensor, a_scales: torch.Tensor, b_scales: torch.Tensor,
                 offsets: torch.Tensor, *, gated: bool = False,
                 out_dtype: torch.dtype = torch.bfloat16,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """``gemm`` of ragged groups: rows ``offsets[e] : offsets[e + 1]`` of ``a [rows, k]`` times
    expert ``e`` of ``b [experts, n or 2n, k]`` (``b_scales [experts, n or 2n]``). ``offsets`` is an
    int32 tensor ``[experts + 1]`` on the device that does not decrease; it is read by the kernel,
    never by the host. Rows that no expert owns are left as they were in ``out`` (and hold anything
    in a result made here)."""
    index = a.get_device()
    if torch.is_grad_enabled() and (a_scales.requires_grad or b_scales.requires_grad
                                    or (out is not None and out.requires_grad)):
        _refuse_gradients()
    refuse_tangents(a_scales, b_scales, out)
    lda, ldb = _codes(a, 2, "a", index), _codes(b, 3, "b", index)
    (rows, k), (experts, width, depth) = a.shape, b.shape
    if depth != k:
        raise ValueError(f"a is {k} deep, b {depth}")
    if rows > MAX_ROWS or width > MAX_ROWS:
        _too_many("a or b", max(rows, width))
    kind = OUT_KINDS.get(out_dtype)
    if kind is None:
        raise ValueError(f"no output in {out_dtype}")
    n = _width(width, gated)
    pa = _vector(a_scales, (rows,), "a_scales", index)
    pb = _vector(b_scales, (experts, width), "b_scales", index)
    if (offsets.dtype is not torch.int32 or offsets.shape != (experts + 1,)
            or not offsets.is_contiguous() or offsets.get_device() != index):
        raise ValueError(f"offsets: expected contiguous int32 {(experts + 1,)} beside the first operand, "
                         f"got {offsets.dtype} {tuple(offsets.shape)} on {offsets.device}")
    _check_device(index)
    if out is None:
        out, ldd = torch.empty(rows, n, dtype=out_dtype, device=a.device), n
    else:
        ldd = _given(out, (rows, n), out_dtype, index, "out")
    _launch(index, "nvfp4_int8_group_gemm", a.data_ptr(), lda, b.data_ptr(), ldb,
            b.stride(0) if experts > 1 else 0, pa, pb, offsets.data_ptr(), out.data_ptr(), ldd, experts,
            rows, n, k, kind, gated)
    return out


def quantize_tokens(x: torch.Tensor, *, rows: torch.Tensor | None = None,
                    out: tuple[torch.Tensor, torch.Tensor] | None = None
                    ) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [tokens, k]`` (FP32, BF16 or FP16) -> INT8 codes and FP32 scales of its rows:
    ``scale = max |x| / 127``, ``code = round(x / scale)`` with ties to even. A zero row has scale
    0; a row with an infinity or a NaN has that as its scale and zero codes. ``rows`` (int32
    ``[R]`` on the device) gathers: row r of the codes is row ``rows[r]`` of ``x``; an index outside
    ``[0, tokens)`` leaves row r as it was. ``out``: codes and scales to write to."""
    index = x.get_device()
    if torch.is_grad_enabled() and (x.requires_grad or (out is not None and out[1].requires_grad)):
        _refuse_gradients()
    refuse_tangents(x, None if out is None else out[1])
    kind = IN_KINDS.get(x.dtype)
    if x.dim() != 2 or kind is None:
        raise ValueError(f"x: expected 2-d FP32, BF16 or FP16, got {x.dtype} {tuple(x.shape)}")
    ldx = _rows(x, x.shape, "x")
    tokens, k = x.shape
    count, source = tokens, None
    if rows is not None:
        if rows.dtype is not torch.int32 or rows.dim() != 1 or not rows.is_contiguous() or rows.get_device() != index:
            raise ValueError(f"rows: expected contiguous 1-d int32 beside the first operand, got {rows.dtype} "
                             f"{tuple(rows.shape)} on {rows.device}")
        count, source = rows.numel(), rows.data_ptr()
    if max(tokens, count, k) > MAX_ROWS:
        _too_many("x", max(tokens, count, k))
    _check_device(index)
    if out is None:
        device = x.device
        ldq = -(-k // 16) * 16
        q = empty_codes(count, k, device)
        scales = torch.empty(count, dtype=torch.float32, device=device)
        ps = scales.data_ptr()
    else:
        q, scales = out
        ldq = _given(q, (count, k), torch.int8, index, "out")
        ps = _vector(scales, (count,), "out", index)
    _launch(index, "nvfp4_int8_quantize", x.data_ptr(), kind, ldx, source, count, tokens, k, q.data_ptr(),
            ldq, ps)
    return q, scales


def residual_norm(x: torch.Tensor, residual: torch.Tensor | None = None, *,
                  post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  residual_scale: float = 1.0, next_weight: torch.Tensor | None = None,
                  eps: float = 1e-6, quantize: bool = False, out_dtype: torch.dtype | None = None,
                  residual_out: torch.Tensor | None = None,
                  out: torch.Tensor | tuple[torch.Tensor, torch.Tensor] | None = None
                  ) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """The end of one block and the start of the next, for ``x [tokens, hidden]``, the block's
    output, and the ``residual`` stream (any of FP32, BF16, FP16 each)::

        p = x / rms(x) * post_weight            (p = x without post_weight)
        r = residual_scale * residual + gate * p
        y = r / rms(r) * next_weight            rms(v) = sqrt(mean(v ** 2) + eps)

    ``residual_scale`` multiplies the residual stream; a factor of the block's output, which some models
    have there, is a ``gate`` that holds it in every element.

    Returns ``(r, y, scales)``: ``r`` in the residual's type, ``y`` (of the unrounded ``r``) in
    ``out_dtype`` (default: the residual's type) or, with ``quantize``, as INT8 codes with their
    ``scales``; what is not made is None. ``gate`` is ``[hidden]`` or ``[gates, hidden]``, each row
    for ``tokens / gates`` consecutive tokens. Weights and gate are FP32, ``eps`` is at least 1e-77.
    Without a residual only ``y = x / rms(x) * next_weight`` is made. ``residual_out`` (may be
    ``residual`` itself) and ``out`` (``y``, or codes and scales) are tensors to write to."""
    index, device = x.get_device(), x.device
    if torch.is_grad_enabled() and (
            x.requires_grad or (residual is not None and residual.requires_grad)
            or (post_weight is not None and post_weight.requires_grad) or (gate is not None and gate.requires_grad)
            or (next_weight is not None and next_weight.requires_grad)
            or (residual_out is not None and residual_out.requires_grad)
            or (out is not None and any(t.requires_grad for t in (out if quantize else (out,))))):
        _refuse_gradients()
    refuse_tangents(x, residual, post_weight, gate, next_weight, residual_out,
                    out[1] if quantize and out is not None else out)
    x_kind = IN_KINDS.get(x.dtype)
    if x.dim() != 2 or x_kind is None:
        raise ValueError(f"x: expected 2-d FP32, BF16 or FP16, got {x.dtype} {tuple(x.shape)}")
    shape = x.shape
    tokens, hidden = shape
    ldx = _rows(x, shape, "x")
    kind, pres, ldres = native.IN_F32, None, 0
    if residual is not None:
        kind = IN_KINDS.get(residual.dtype)
        if kind is None or residual.shape != shape or residual.get_device() != index:
            raise ValueError(f"residual: expected {tuple(shape)} beside the first operand, got "
                             f"{residual.dtype} {tuple(residual.shape)} on {residual.device}")
        pres, ldres = residual.data_ptr(), _rows(residual, shape, "residual")
    elif residual_out is not None or post_weight is not None or gate is not None or residual_scale != 1.0:
        raise ValueError("without a residual there is only the norm of x: no post_weight, gate, residual_scale "
                         "or residual_out")
    if next_weight is None and (residual is None or quantize or out_dtype is not None):
        raise ValueError("next_weight is missing: there is nothing to norm, quantise or return")
    if quantize and out_dtype is not None:
        raise ValueError("codes have no out_dtype")
    if out is not None and next_weight is None:
        raise ValueError("out without next_weight")
    if tokens > MAX_ROWS:
        _too_many("x", tokens)
    if hidden > MAX_HIDDEN:
        raise ValueError(f"rows of {hidden}, at most {MAX_HIDDEN}")
    row = (hidden,)
    ppost = None if post_weight is None else _vector(post_weight, row, "post_weight", index)
    pnext = None if next_weight is None else _vector(next_weight, row, "next_weight", index)
    pgate, gates = None, 0
    if gate is not None:
        gates = gate.shape[0] if gate.dim() == 2 else 1
        if gates == 0 or tokens % gates:  # the address of no rows is null, which is no gate
            raise ValueError(f"{tokens} tokens do not share {gates} gates evenly")
        pgate = _vector(gate, (gates, hidden) if gate.dim() == 2 else row, "gate", index)
    _check_device(index)
    r, pr, ldr = None, None, 0
    if residual is not None:
        if residual_out is None:
            r, ldr = torch.empty(tokens, hidden, dtype=residual.dtype, device=device), hidden
        else:
            r, ldr = residual_out, _given(residual_out, shape, residual.dtype, index, "residual_out")
        pr = r.data_ptr()
    y, py, ldy, y_kind, scales, pscales = None, None, 0, native.NORM_CODES, None, None
    if next_weight is not None:
        if quantize:
            if out is None:
                y, ldy = empty_codes(tokens, hidden, device), -(-hidden // 16) * 16
                scales = torch.empty(tokens, dtype=torch.float32, device=device)
                pscales = scales.data_ptr()
            else:
                y, scales = out
                ldy = _given(y, shape, torch.int8, index, "out")
                pscales = _vector(scales, (tokens,), "out", index)
        else:
            dtype = out_dtype or (x if residual is None else residual).dtype
            y_kind = IN_KINDS.get(dtype)
            if y_kind is None:
                raise ValueError(f"no output in {dtype}")
            if out is None:
                y, ldy = torch.empty(tokens, hidden, dtype=dtype, device=device), hidden
            else:
                y, ldy = out, _given(out, shape, dtype, index, "out")
        py = y.data_ptr()
    _launch(index, "nvfp4_residual_norm", x.data_ptr(), x_kind, ldx, pres, kind, ldres, ppost, pgate, gates,
            residual_scale, pnext, eps, pr, ldr, py, y_kind, ldy, pscales, tokens, hidden)
    return r, y, scales
