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
compute capability 10.0 ``RuntimeError``. There is no backward: operands that require a gradient
are refused while gradients are recorded.

Codes are ``torch.int8`` ``[rows, k]`` whose rows start 16-byte aligned and a multiple of 16 bytes
apart, which is what ``quantize_tokens`` and ``residual_norm`` return for every ``k`` (a view of
padded rows where ``k`` is no multiple of 16; ``empty_codes`` makes such a buffer). Scales are FP32
and contiguous. Weights are quantised by the same function, a scale for each output channel:
``quantize_tokens(w)``.
"""

from __future__ import annotations

import contextlib

import torch

from . import native

OUT_KINDS = {torch.float16: native.OUT_F16, torch.float32: native.OUT_F32,
             torch.bfloat16: native.OUT_BF16}
IN_KINDS = {torch.float32: native.IN_F32, torch.bfloat16: native.IN_BF16,
            torch.float16: native.IN_F16}
MAX_DEPTH = 131071  # k: sums of products of codes stay within 32 bits
MAX_EXPERTS = 1024
MAX_HIDDEN = 32768

_supported: dict[int, bool] = {}


def _launch_on(device: torch.device):
    """(context that makes ``device`` current, its current stream)."""
    if device.type != "cuda":
        raise RuntimeError(f"sm_100a code cannot run on {device}")
    index = device.index
    if index not in _supported:
        _supported[index] = native.device_supported(index)
    if not _supported[index]:
        raise RuntimeError(f"sm_100a code cannot run on {device}")
    stream = torch.cuda.current_stream(device).cuda_stream
    if index == torch.cuda.current_device():
        return contextlib.nullcontext(), stream
    return torch.cuda.device(device), stream


def _refuse_gradients(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("the INT8 operators have no backward; call them under torch.no_grad()")


def _pitch(t: torch.Tensor, what: str) -> int:
    """Elements between the rows of ``t`` (its last but one dimension)."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}: elements of a row must be neighbours")
    if t.shape[-2] > 1:
        return t.stride(-2)
    return -(-t.shape[-1] // 16) * 16  # one row: nothing lies between


def _vector(t: torch.Tensor, shape: tuple, what: str, device: torch.device) -> int:
    if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{what}: expected contiguous float32 {shape} on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def empty_codes(rows: int, k: int, device: torch.device | str) -> torch.Tensor:
    """An INT8 ``[rows, k]`` buffer whose rows lie 16-byte aligned."""
    pitch = -(-k // 16) * 16
    codes = torch.empty((rows, pitch), dtype=torch.int8, device=device)
    return codes if pitch == k else codes[:, :k]


def _codes(t: torch.Tensor, dims: int, what: str, device: torch.device) -> int:
    if t.dtype != torch.int8 or t.dim() != dims or t.device != device:
        raise ValueError(f"{what}: expected {dims}-d int8 on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return _pitch(t, what)


def _output(out: torch.Tensor | None, rows: int, n: int, dtype: torch.dtype, device: torch.device):
    """(tensor, elements between its rows)"""
    if out is None:
        return torch.empty((rows, n), dtype=dtype, device=device), n
    if out.dtype != dtype or tuple(out.shape) != (rows, n) or out.device != device:
        raise ValueError(f"out: expected {dtype} {(rows, n)} on {device}, got {out.dtype} "
                         f"{tuple(out.shape)} on {out.device}")
    return out, _pitch(out, "out")


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
    ``silu(gate) * up`` ``[m, n]``. ``out``: a tensor to write it to."""
    device = a.device
    _refuse_gradients(a_scales, b_scales, bias, out)
    lda, ldb = _codes(a, 2, "a", device), _codes(b, 2, "b", device)
    (m, k), (width, depth) = a.shape, b.shape
    if depth != k:
        raise ValueError(f"a is {k} deep, b {depth}")
    if out_dtype not in OUT_KINDS:
        raise ValueError(f"no output in {out_dtype}")
    n = _width(width, gated)
    pa, pb = _vector(a_scales, (m,), "a_scales", device), _vector(b_scales, (width,), "b_scales", device)
    pbias = None if bias is None else _vector(bias, (width,), "bias", device)
    current, stream = _launch_on(device)
    out, ldd = _output(out, m, n, out_dtype, device)
    with current:
        native.check(native.load().nvfp4_int8_gemm(
            a.data_ptr(), lda, b.data_ptr(), ldb, pa, pb, pbias, out.data_ptr(), ldd, m, n, k,
            OUT_KINDS[out_dtype], gated, stream))
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
    device = a.device
    _refuse_gradients(a_scales, b_scales, out)
    lda, ldb = _codes(a, 2, "a", device), _codes(b, 3, "b", device)
    (rows, k), (experts, width, depth) = a.shape, b.shape
    if depth != k:
        raise ValueError(f"a is {k} deep, b {depth}")
    if out_dtype not in OUT_KINDS:
        raise ValueError(f"no output in {out_dtype}")
    n = _width(width, gated)
    pa = _vector(a_scales, (rows,), "a_scales", device)
    pb = _vector(b_scales, (experts, width), "b_scales", device)
    if (offsets.dtype != torch.int32 or tuple(offsets.shape) != (experts + 1,)
            or not offsets.is_contiguous() or offsets.device != device):
        raise ValueError(f"offsets: expected contiguous int32 {(experts + 1,)} on {device}, got "
                         f"{offsets.dtype} {tuple(offsets.shape)} on {offsets.device}")
    current, stream = _launch_on(device)
    out, ldd = _output(out, rows, n, out_dtype, device)
    with current:
        native.check(native.load().nvfp4_int8_group_gemm(
            a.data_ptr(), lda, b.data_ptr(), ldb, b.stride(0) if experts > 1 else 0, pa, pb,
            offsets.data_ptr(), out.data_ptr(), ldd, experts, rows, n, k, OUT_KINDS[out_dtype],
            gated, stream))
    return out


def quantize_tokens(x: torch.Tensor, *, rows: torch.Tensor | None = None,
                    out: tuple[torch.Tensor, torch.Tensor] | None = None
                    ) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [tokens, k]`` (FP32, BF16 or FP16) -> INT8 codes and FP32 scales of its rows:
    ``scale = max |x| / 127``, ``code = round(x / scale)`` with ties to even. A zero row has scale
    0; a row with an infinity or a NaN has that as its scale and zero codes. ``rows`` (int32
    ``[R]`` on the device) gathers: row r of the codes is row ``rows[r]`` of ``x``; an index outside
    ``[0, tokens)`` leaves row r as it was. ``out``: codes and scales to write to."""
    device = x.device
    _refuse_gradients(x)
    if x.dim() != 2 or x.dtype not in IN_KINDS:
        raise ValueError(f"x: expected 2-d FP32, BF16 or FP16, got {x.dtype} {tuple(x.shape)}")
    ldx = _pitch(x, "x")
    tokens, k = x.shape
    count, source = tokens, None
    if rows is not None:
        if rows.dtype != torch.int32 or rows.dim() != 1 or not rows.is_contiguous() or rows.device != device:
            raise ValueError(f"rows: expected contiguous 1-d int32 on {device}, got {rows.dtype} "
                             f"{tuple(rows.shape)} on {rows.device}")
        count, source = rows.numel(), rows.data_ptr()
    current, stream = _launch_on(device)
    if out is None:
        q = empty_codes(count, k, device)
        scales = torch.empty((count,), dtype=torch.float32, device=device)
    else:
        q, scales = out
        if tuple(q.shape) != (count, k):
            raise ValueError(f"out: expected codes {(count, k)}, got {tuple(q.shape)}")
    ldq = _codes(q, 2, "out", device)
    ps = _vector(scales, (count,), "out", device)
    with current:
        native.check(native.load().nvfp4_int8_quantize(
            x.data_ptr(), IN_KINDS[x.dtype], ldx, source, count, tokens, k, q.data_ptr(), ldq, ps,
            stream))
    return q, scales


def residual_norm(x: torch.Tensor, residual: torch.Tensor | None = None, *,
                  post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  residual_scale: float = 1.0, next_weight: torch.Tensor | None = None,
                  eps: float = 1e-6, quantize: bool = False, out_dtype: torch.dtype | None = None,
                  residual_out: torch.Tensor | None = None
                  ) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """The end of one block and the start of the next, for ``x [tokens, hidden]``, the block's
    output, and the ``residual`` stream (any of FP32, BF16, FP16 each)::

        p = x / rms(x) * post_weight            (p = x without post_weight)
        r = residual_scale * residual + gate * p
        y = r / rms(r) * next_weight            rms(v) = sqrt(mean(v ** 2) + eps)

    Returns ``(r, y, scales)``: ``r`` in the residual's type, ``y`` (of the unrounded ``r``) in
    ``out_dtype`` (default: the residual's type) or, with ``quantize``, as INT8 codes with their
    ``scales``; what is not made is None. ``gate`` is ``[hidden]`` or ``[gates, hidden]``, each row
    for ``tokens / gates`` consecutive tokens. Weights and gate are FP32. Without a residual only
    ``y = x / rms(x) * next_weight`` is made. ``residual_out`` may be ``residual`` itself."""
    device = x.device
    _refuse_gradients(x, residual, post_weight, gate, next_weight)
    if x.dim() != 2 or x.dtype not in IN_KINDS:
        raise ValueError(f"x: expected 2-d FP32, BF16 or FP16, got {x.dtype} {tuple(x.shape)}")
    tokens, hidden = x.shape
    ldx = _pitch(x, "x")
    kind, pres, ldres = native.IN_F32, None, 0
    if residual is not None:
        if residual.dtype not in IN_KINDS or residual.shape != x.shape or residual.device != device:
            raise ValueError(f"residual: expected {tuple(x.shape)} on {device}, got "
                             f"{residual.dtype} {tuple(residual.shape)} on {residual.device}")
        kind, pres, ldres = IN_KINDS[residual.dtype], residual.data_ptr(), _pitch(residual, "residual")
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    if next_weight is None and (residual is None or quantize or out_dtype is not None):
        raise ValueError("next_weight is missing: there is nothing to norm, quantise or return")
    if quantize and out_dtype is not None:
        raise ValueError("codes have no out_dtype")
    ppost = None if post_weight is None else _vector(post_weight, (hidden,), "post_weight", device)
    pnext = None if next_weight is None else _vector(next_weight, (hidden,), "next_weight", device)
    pgate, gates = None, 0
    if gate is not None:
        gates = gate.shape[0] if gate.dim() == 2 else 1
        pgate = _vector(gate, (gates, hidden) if gate.dim() == 2 else (hidden,), "gate", device)
    current, stream = _launch_on(device)
    r, pr, ldr = None, None, 0
    if residual is not None:
        r, ldr = _output(residual_out, tokens, hidden, residual.dtype, device)
        pr = r.data_ptr()
    y, py, ldy, y_kind, scales, pscales = None, None, 0, native.NORM_CODES, None, None
    if next_weight is not None:
        if quantize:
            y = empty_codes(tokens, hidden, device)
            ldy = -(-hidden // 16) * 16
            scales = torch.empty((tokens,), dtype=torch.float32, device=device)
            pscales = scales.data_ptr()
        else:
            dtype = out_dtype or (x if residual is None else residual).dtype
            if dtype not in IN_KINDS:
                raise ValueError(f"no output in {dtype}")
            y, ldy, y_kind = torch.empty((tokens, hidden), dtype=dtype, device=device), hidden, IN_KINDS[dtype]
        py = y.data_ptr()
    with current:
        native.check(native.load().nvfp4_residual_norm(
            x.data_ptr(), IN_KINDS[x.dtype], ldx, pres, kind, ldres, ppost, pgate, gates,
            residual_scale, pnext, eps, pr, ldr, py, y_kind, ldy, pscales, tokens, hidden, stream))
    return r, y, scales
