"""Workloads of the 8-bit-integer path (``harness.int8``): the product with a scale for each
token and channel, the same over ragged groups, the per-token quantiser and the norms around a
block. No counterpart in the reference, whose 8-bit products are FP8; shapes come from the
``harness.models`` table and from sizes that are odd on purpose.

References are torch operations; integers are summed in FP64, which holds them exactly."""

from __future__ import annotations

import torch

from .. import int8
from ..registry import register
from ..throughput import model_case, skewed_lengths
from ..workload import CaseSpec, Workload

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def make_codes(workload: Workload, generator: torch.Generator, *shape: int) -> torch.Tensor:
    """Uniform INT8 codes, -128 included, in rows padded to 16 bytes."""
    *lead, k = shape
    pitch = -(-k // 16) * 16
    return torch.randint(-128, 128, (*lead, pitch), dtype=torch.int8, device=workload.device,
                         generator=generator)[..., :k]


def scaled_product(a, b, a_scales, b_scales, bias=None, gated=False, dtype=torch.float32):
    """``int8.gemm`` in torch: exact sums, then the kernel's order of FP32 operations."""
    y = (a.double() @ b.double().T).float() * a_scales[:, None] * b_scales
    if bias is not None:
        y = y + bias
    if gated:
        gate, up = y.chunk(2, dim=1)
        y = torch.nn.functional.silu(gate) * up
    return y.to(dtype)


def quantized(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``int8.quantize_tokens`` in torch (divisors as tensors: torch multiplies by the reciprocal
    of a Python number)."""
    x = x.float()
    scales = x.abs().amax(1) / torch.full((), 127.0, device=x.device)
    live = torch.isfinite(scales) & (scales > 0)
    codes = (x / torch.where(live, scales, torch.ones_like(scales))[:, None]).round().clamp(-127, 127)
    return torch.where(live[:, None], codes, torch.zeros_like(codes)).to(torch.int8), scales


def rms_normed(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """FP32 ``x / rms(x) * weight``, the statistic in FP64 as the kernel takes it."""
    mean = x.double().square().sum(1, keepdim=True) / x.shape[1]
    return x * (1 / (mean + eps).sqrt()).float() * weight


class Int8Workload(Workload):
    """``run`` calls the function of ``harness.int8`` on the workload's device; nothing is kept
    between calls, so there is no plan or workspace to prepare, only the outputs."""

    def call(self, inputs: tuple, outputs: tuple | None = None) -> tuple:
        """The outputs of ``inputs``, new ones or those given."""
        raise NotImplementedError

    def run(self, inputs):
        self._check_open()
        self._check_supported()
        return self.call(inputs)

    def prepare(self, inputs):
        outputs = self.run(inputs)

        def launch() -> tuple:
            self._check_open()
            self.call(inputs, outputs)
            return outputs

        return launch, outputs

    def check_status(self) -> None:
        int8.check_status(self.device)


@register(name="int8_gemm", supported_arches=("sm_100a",))
class Int8GEMM(Int8Workload):
    """``D = (A B^T) * a_scales * b_scales + bias``, or the gated pair. Inputs
    ``(a, b, a_scales, b_scales, bias or None, gated, out dtype)``."""

    entry_point = "nvfp4_int8_gemm"

    def get_cases(self):
        cases = []
        for seed, (m, n, k, gated, bias, out) in enumerate((
                (1, 64, 16, False, False, "bf16"), (1, 1, 1, False, False, "fp32"),
                (37, 129, 100, False, True, "fp16"), (130, 72, 640, True, False, "bf16"),
                (257, 200, 2064, False, False, "fp32"), (300, 515, 48, True, True, "fp16"))):
            cases.append(CaseSpec(f"m{m}_n{n}_k{k}_{out}" + "_gated" * gated + "_bias" * bias,
                                  dict(m=m, n=n, k=k, gated=gated, bias=bias, out=out), seed))
        for model in ("llama3_70b", "qwen3_32b"):
            from ..models import MODELS

            shapes = MODELS[model].linear_shapes()
            for tokens in (1, 64, 4096):
                for layer in ("o", "gate_up", "down"):
                    n, k = shapes[layer]
                    gated = layer == "gate_up"
                    cases.append(model_case(
                        f"{model}_{layer}_t{tokens}",
                        dict(m=tokens, n=n // 2 if gated else n, k=k, gated=gated, bias=False,
                             out="bf16"), model, layer))
        return cases

    def get_inputs(self, case):
        p, g = case.params, self.generator(case)
        width = p["n"] * (2 if p["gated"] else 1)
        a, b = make_codes(self, g, p["m"], p["k"]), make_codes(self, g, width, p["k"])
        scale = 0.02 / p["k"] ** 0.5
        sa = 0.5 + torch.rand(p["m"], device=self.device, generator=g)
        sb = scale * (0.5 + torch.rand(width, device=self.device, generator=g))
        bias = self.randn((width,), g, torch.float32) if p["bias"] else None
        return a, b, sa, sb, bias, p["gated"], DTYPES[p["out"]]

    def get_reference(self, inputs):
        return (scaled_product(*inputs),)

    def call(self, inputs, outputs=None):
        a, b, sa, sb, bias, gated, dtype = inputs
        return (int8.gemm(a, b, sa, sb, bias=bias, gated=gated, out_dtype=dtype,
                          out=outputs and outputs[0]),)

    def validate(self, ref, impl):
        # The same exact sums; a rounding of the output type, and in the gate FP32 ones.
        eps = torch.finfo(ref[0].dtype).eps
        self.assert_close(ref, impl, rtol=eps + 1e-5, atol=1e-6)


@register(name="int8_group_gemm", supported_arches=("sm_100a",))
class Int8GroupGEMM(Int8Workload):
    """The product over ragged groups. Inputs
    ``(a, b, a_scales, b_scales, offsets, gated, out dtype)``."""

    entry_point = "nvfp4_int8_group_gemm"

    def get_cases(self):
        def case(counts, n, k, gated, out, seed):
            return CaseSpec(f"g{len(counts)}_rows{sum(counts)}_n{n}_k{k}_{out}" + "_gated" * gated,
                            dict(counts=list(counts), n=n, k=k, gated=gated, out=out), seed)

        cases = [case((1,), 8, 16, False, "fp32", 1), case((0, 3, 0, 130, 1), 72, 100, False, "fp16", 2),
                 case((5, 0, 300, 64), 136, 528, True, "bf16", 3),
                 case(skewed_lengths(700, 24, seed=4, sigma=1.5, minimum=0), 40, 256, True, "fp32", 4)]
        for tokens in (16, 1024):
            for layer, gated in (("expert_gate_up", True), ("expert_down", False)):
                from ..models import MODELS

                spec, local = MODELS["deepseek_v3"], 32
                n, k = spec.linear_shapes()[layer]
                counts = skewed_lengths(tokens * spec.top_k * local // spec.experts, local,
                                        seed=tokens, minimum=0)
                cases.append(model_case(f"deepseek_v3_{layer}_t{tokens}",
                                        dict(counts=counts, n=n // 2 if gated else n, k=k,
                                             gated=gated, out="bf16"), "deepseek_v3", layer))
        return cases

    def get_inputs(self, case):
        p, g = case.params, self.generator(case)
        counts, width = p["counts"], p["n"] * (2 if p["gated"] else 1)
        rows = sum(counts)
        a, b = make_codes(self, g, rows, p["k"]), make_codes(self, g, len(counts), width, p["k"])
        sa = 0.5 + torch.rand(rows, device=self.device, generator=g)
        sb = 0.02 / p["k"] ** 0.5 * (0.5 + torch.rand((len(counts), width), device=self.device, generator=g))
        offsets = torch.tensor([0, *counts], dtype=torch.int32).cumsum(0, dtype=torch.int32)
        return a, b, sa, sb, offsets.to(self.device), p["gated"], DTYPES[p["out"]]

    def get_reference(self, inputs):
        a, b, sa, sb, offsets, gated, dtype = inputs
        edges = offsets.tolist()
        return (torch.cat([
            scaled_product(a[lo:hi], b[e], sa[lo:hi], sb[e], None, gated, dtype)
            for e, (lo, hi) in enumerate(zip(edges, edges[1:]))]),)

    def call(self, inputs, outputs=None):
        a, b, sa, sb, offsets, gated, dtype = inputs
        return (int8.grouped_gemm(a, b, sa, sb, offsets, gated=gated, out_dtype=dtype,
                                  out=outputs and outputs[0]),)

    validate = Int8GEMM.validate


@register(name="int8_quantize", supported_arches=("sm_100a",))
class Int8Quantize(Int8Workload):
    """Rows -> INT8 codes and scales; inputs ``(x, rows or None)``."""

    entry_point = "nvfp4_int8_quantize"

    def get_cases(self):
        return [CaseSpec(f"t{tokens}_k{k}_{kind}" + (f"_r{rows}" if rows else ""),
                         dict(tokens=tokens, k=k, kind=kind, rows=rows), seed)
                for seed, (tokens, k, kind, rows) in enumerate((
                    (1, 1, "fp32", 0), (1, 7168, "bf16", 0), (33, 100, "fp16", 0),
                    (5, 2880, "fp32", 40), (130, 8200, "bf16", 7), (2, 16385, "fp16", 0)))]

    def get_inputs(self, case):
        p, g = case.params, self.generator(case)
        x = self.randn((p["tokens"], p["k"]), g, DTYPES[p["kind"]], scale=3.0)
        x[0] = 0
        rows = torch.randint(0, p["tokens"], (p["rows"],), dtype=torch.int32, device=self.device,
                             generator=g) if p["rows"] else None
        return x, rows

    def get_reference(self, inputs):
        x, rows = inputs
        return quantized(x if rows is None else x[rows.long()])

    def call(self, inputs, outputs=None):
        return int8.quantize_tokens(inputs[0], rows=inputs[1], out=outputs)

    def validate(self, ref, impl):
        # Both quotients are correctly rounded: the same codes and scales, bit for bit.
        self.assert_close(ref, impl, rtol=0, atol=0)


@register(name="residual_norm", supported_arches=("sm_100a",))
class ResidualNorm(Int8Workload):
    """The norms around a block. Inputs ``(x, residual, post_weight, gate, residual scale,
    next_weight, eps, quantize)``; outputs: those that are made."""

    entry_point = "nvfp4_residual_norm"

    def get_cases(self):
        return [CaseSpec(f"t{tokens}_h{hidden}_{x}_{residual}_g{gates}" + "_post" * post + "_codes" * codes,
                         dict(tokens=tokens, hidden=hidden, x=x, residual=residual, gates=gates,
                              post=post, codes=codes), seed)
                for seed, (tokens, hidden, x, residual, gates, post, codes) in enumerate((
                    (1, 1, "fp32", "fp32", 0, True, False), (1, 7168, "fp32", "bf16", 1, True, True),
                    (33, 100, "fp16", "fp16", 0, False, False), (12, 2880, "bf16", "bf16", 3, True, False),
                    (130, 5120, "bf16", "fp32", 130, True, True), (3, 16385, "fp16", "bf16", 1, False, True)))]

    def get_inputs(self, case):
        p, g = case.params, self.generator(case)
        shape = (p["tokens"], p["hidden"])
        weight = lambda: 0.5 + torch.rand(p["hidden"], device=self.device, generator=g)  # noqa: E731
        x = self.randn(shape, g, DTYPES[p["x"]], scale=3.0)
        residual = self.randn(shape, g, DTYPES[p["residual"]])
        gate = self.randn((p["gates"], p["hidden"]), g, torch.float32) if p["gates"] else None
        return x, residual, weight() if p["post"] else None, gate, 0.5, weight(), 1e-6, p["codes"]

    def get_reference(self, inputs):
        x, residual, post, gate, scale, weight, eps, codes = inputs
        p = x.float()
        if post is not None:
            p = rms_normed(p, post, eps)
        if gate is not None:
            p = p * gate.repeat_interleave(x.shape[0] // gate.shape[0], dim=0)
        r = residual.float() * scale + p
        y = rms_normed(r, weight, eps)
        return (r.to(residual.dtype), *quantized(y)) if codes else (r.to(residual.dtype), y.to(residual.dtype))

    def call(self, inputs, outputs=None):
        x, residual, post, gate, scale, weight, eps, codes = inputs
        r, y = (None, None) if outputs is None else (outputs[0], outputs[1:] if codes else outputs[1])
        made = int8.residual_norm(x, residual, post_weight=post, gate=gate, residual_scale=scale,
                                  next_weight=weight, eps=eps, quantize=codes, residual_out=r, out=y)
        return tuple(t for t in made if t is not None)

    def validate(self, ref, impl):
        # The kernel keeps the reference's order of roundings: the same bits, codes included.
        self.assert_close(ref, impl, rtol=0, atol=0)
