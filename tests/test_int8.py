"""The 8-bit-integer operators without a GPU: what the functions of ``harness.int8`` and the C
entry points refuse, before anything is launched, and the torch references of their workloads
against the definitions in 64 bits."""

import numpy as np
import pytest
import torch

from harness import get_workload, int8, native
from harness.workloads import int8 as references


@pytest.fixture(scope="module")
def library():
    if not native.LIBRARY_PATH.is_file():
        from harness import build
        build.build()
    return native.load()


def codes(*shape):
    return torch.zeros(shape, dtype=torch.int8)


def ones(*shape):
    return torch.ones(shape)


def test_functions_refuse_what_they_cannot_take():
    """Every refusal is a ValueError of the host; what passes the checks ends at the device, which
    is none here."""
    a, b, sa, sb = codes(3, 32), codes(8, 32), ones(3), ones(8)
    for call in (
        lambda: int8.gemm(a, codes(8, 48), sa, sb),                       # depths differ
        lambda: int8.gemm(a.float(), b, sa, sb),                          # not codes
        lambda: int8.gemm(a, b, ones(4), sb),                             # a scale too many
        lambda: int8.gemm(a, b, sa.half(), sb),
        lambda: int8.gemm(a, b, sa, ones(16)[::2]),
        lambda: int8.gemm(a, codes(7, 32), sa, ones(7), gated=True),      # an odd pair
        lambda: int8.gemm(a, b, sa, sb, bias=ones(4)),
        lambda: int8.gemm(a, b, sa, sb, out_dtype=torch.float64),
        lambda: int8.gemm(codes(32, 3).T, b, sa, sb),                     # columns, not rows
        lambda: int8.gemm(a, b, sa.clone().requires_grad_(), sb),
        lambda: int8.grouped_gemm(a, codes(2, 8, 32), sa, ones(2, 8), torch.zeros(3, dtype=torch.int64)),
        lambda: int8.grouped_gemm(a, codes(2, 8, 32), sa, ones(2, 8), torch.zeros(2, dtype=torch.int32)),
        lambda: int8.grouped_gemm(a, codes(2, 8, 32), sa, ones(16), torch.zeros(3, dtype=torch.int32)),
        lambda: int8.gemm(codes(1, 16).expand((1 << 30) + 1, 16), b[:, :16], sa, sb),   # too many rows
        lambda: int8.quantize_tokens(ones(1, 1).expand(1 << 32, 1)),
        lambda: int8.residual_norm(ones(1, 1).expand(1 << 32, 1), next_weight=ones(1)),
        lambda: int8.residual_norm(ones(1, 32769), next_weight=ones(32769)),
        lambda: int8.quantize_tokens(ones(4)),
        lambda: int8.quantize_tokens(ones(4, 4).double()),
        lambda: int8.quantize_tokens(ones(4, 4).T[:, ::2]),
        lambda: int8.quantize_tokens(ones(4, 4), rows=torch.zeros(4, dtype=torch.int64)),
        lambda: int8.residual_norm(ones(4, 8)),                           # nothing to make
        lambda: int8.residual_norm(ones(4, 8), ones(4, 9), next_weight=ones(8)),
        lambda: int8.residual_norm(ones(4, 8), ones(4, 8), post_weight=ones(9)),
        lambda: int8.residual_norm(ones(4, 8), ones(4, 8), gate=ones(2, 9), next_weight=ones(8)),
        lambda: int8.residual_norm(ones(4, 8), ones(4, 8), quantize=True),
        lambda: int8.residual_norm(ones(4, 8), ones(4, 8), next_weight=ones(8), quantize=True,
                                   out_dtype=torch.float16),
        lambda: int8.residual_norm(ones(4, 8), next_weight=ones(8), residual_out=ones(4, 8)),
        lambda: int8.residual_norm(ones(4, 8), next_weight=ones(8), out=ones(4, 8).requires_grad_()),
        lambda: int8.quantize_tokens(ones(4, 16), out=(codes(4, 16), ones(4).requires_grad_())),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: int8.gemm(a, b, sa, sb),
                 lambda: int8.quantize_tokens(ones(4, 4)),
                 lambda: int8.residual_norm(ones(4, 8), next_weight=ones(8))):
        with pytest.raises(RuntimeError):
            call()


def test_entry_points_refuse_before_cuda(library):
    """Addresses here are never followed: each call is wrong in one argument."""
    def gemm(a=16, lda=32, b=32, ldb=32, sa=16, sb=16, bias=None, d=16, ldd=8, m=4, n=8, k=32, out=0):
        return library.nvfp4_int8_gemm(a, lda, b, ldb, sa, sb, bias, d, ldd, m, n, k, out, 0, None)

    assert gemm(a=None) == native.E_INVALID_ARGUMENT
    assert gemm(d=None) == native.E_INVALID_ARGUMENT
    assert gemm(out=7) == native.E_INVALID_ARGUMENT
    assert gemm(lda=16) == native.E_INVALID_ARGUMENT
    assert gemm(ldb=0) == native.E_INVALID_ARGUMENT
    assert gemm(ldd=4) == native.E_INVALID_ARGUMENT
    assert gemm(m=-1) == native.E_UNSUPPORTED_SHAPE
    assert gemm(n=0) == native.E_UNSUPPORTED_SHAPE
    assert gemm(m=(1 << 30) + 1) == native.E_UNSUPPORTED_SHAPE
    assert gemm(n=(1 << 30) + 1, ldd=1 << 31) == native.E_UNSUPPORTED_SHAPE
    assert gemm(k=0) == native.E_UNSUPPORTED_SHAPE
    assert gemm(k=131072, lda=131072, ldb=131072) == native.E_UNSUPPORTED_SHAPE
    assert gemm(a=24) == native.E_MISALIGNED
    assert gemm(lda=40) == native.E_MISALIGNED
    assert gemm(sa=18) == native.E_MISALIGNED
    assert gemm(bias=2) == native.E_MISALIGNED
    assert gemm(d=18, out=native.OUT_F32) == native.E_MISALIGNED
    assert gemm(m=0, a=None) == 0

    def grouped(offsets=16, experts=2, stride=256, rows=4):
        return library.nvfp4_int8_group_gemm(16, 32, 16, 32, stride, 16, 16, offsets, 16, 8, experts,
                                             rows, 8, 32, 0, 0, None)

    assert grouped(offsets=None) == native.E_INVALID_ARGUMENT
    assert grouped(experts=0) == native.E_UNSUPPORTED_SHAPE
    assert grouped(experts=1025) == native.E_UNSUPPORTED_SHAPE
    assert grouped(stride=-256) == native.E_INVALID_ARGUMENT
    assert grouped(stride=240) == native.E_INVALID_ARGUMENT      # experts overlap
    assert grouped(stride=264) == native.E_MISALIGNED
    assert grouped(offsets=18) == native.E_MISALIGNED
    assert grouped(rows=0) == 0

    def quantize(x=16, kind=0, ldx=8, source=None, rows=4, tokens=4, k=8, q=16, ldq=16, scales=16):
        return library.nvfp4_int8_quantize(x, kind, ldx, source, rows, tokens, k, q, ldq, scales, None)

    assert quantize(x=None) == native.E_INVALID_ARGUMENT
    assert quantize(kind=3) == native.E_INVALID_ARGUMENT
    assert quantize(rows=5) == native.E_INVALID_ARGUMENT
    assert quantize(ldx=0) == native.E_INVALID_ARGUMENT
    assert quantize(ldq=4) == native.E_INVALID_ARGUMENT
    assert quantize(k=0) == native.E_UNSUPPORTED_SHAPE
    assert quantize(x=18) == native.E_MISALIGNED
    assert quantize(rows=0, tokens=0) == 0

    def norm(x=16, residual=16, r=16, post=None, gate=None, gates=0, scale=1.0, weight=16, eps=1e-6,
             y=16, y_kind=0, scales=None, tokens=4, hidden=8, ldx=8, ldr=8):
        return library.nvfp4_residual_norm(x, 0, ldx, residual, 0, 8, post, gate, gates, scale, weight,
                                           eps, r, ldr, y, y_kind, 8, scales, tokens, hidden, None)

    assert norm(x=None) == native.E_INVALID_ARGUMENT
    assert norm(r=None) == native.E_INVALID_ARGUMENT
    assert norm(y=None) == native.E_INVALID_ARGUMENT
    assert norm(y_kind=native.NORM_CODES) == native.E_INVALID_ARGUMENT
    assert norm(y_kind=5) == native.E_INVALID_ARGUMENT
    assert norm(eps=0.0) == native.E_INVALID_ARGUMENT
    assert norm(eps=float("nan")) == native.E_INVALID_ARGUMENT
    assert norm(residual=None, r=None, post=16) == native.E_INVALID_ARGUMENT
    assert norm(residual=None, r=None, scale=0.5) == native.E_INVALID_ARGUMENT
    assert norm(ldx=4) == native.E_INVALID_ARGUMENT
    assert norm(ldr=0) == native.E_INVALID_ARGUMENT
    assert norm(gate=16, gates=3) == native.E_UNSUPPORTED_SHAPE
    assert norm(hidden=32769) == native.E_UNSUPPORTED_SHAPE
    assert norm(x=18) == native.E_MISALIGNED
    assert norm(tokens=0, x=None) == 0

    assert library.nvfp4_moe_offsets(None, 4, 16, None) == native.E_INVALID_ARGUMENT
    assert library.nvfp4_moe_offsets(16, 0, 16, None) == native.E_UNSUPPORTED_SHAPE
    assert library.nvfp4_moe_place_offsets(16, 1, 8, 2, 4, None, 8, 16, 16, 16, None) == \
        native.E_INVALID_ARGUMENT
    assert library.nvfp4_moe_place_offsets(16, 1, 8, 2, 4, 16, 7, 16, 16, 16, None) == \
        native.E_INVALID_ARGUMENT      # fewer rows than pairs


def test_workloads_are_registered_with_cases():
    for name in ("int8_gemm", "int8_group_gemm", "int8_quantize", "residual_norm"):
        workload = get_workload(name)(None, device="cpu")
        cases = workload.get_cases()
        assert len({c.name for c in cases}) == len(cases) > 3
        case = cases[1]
        inputs = workload.get_inputs(case)
        reference = workload.get_reference(inputs)
        workload.validate(reference, workload.get_reference(workload.get_inputs(case)))
        with pytest.raises(RuntimeError):
            workload.run(inputs)


def test_quantiser_reference_is_the_definition():
    """Scale and codes by numpy's correctly rounded FP32 division."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((9, 50)) * rng.lognormal(0, 3, (9, 1))).astype(np.float32)
    x[2] = 0
    x[4, 7] = np.inf
    x[5, 3] = np.nan
    x[6] = 1e-45
    q, s = references.quantized(torch.from_numpy(x))
    for row, codes_, scale in zip(x, q.numpy(), s.numpy()):
        amax = np.abs(row).max()
        want = np.float32(amax) / np.float32(127)
        np.testing.assert_array_equal(scale, want)
        if want > 0 and np.isfinite(want):
            np.testing.assert_array_equal(codes_, np.clip(np.rint(row / want), -127, 127))
        else:
            assert not codes_.any()


def test_combine_of_fp32_rows_refuses_before_cuda(library):
    def combine(y=16, rows=16, weights=16, out=16, tokens=4, choices=2, hidden=16):
        return library.nvfp4_moe_combine_f32(y, rows, weights, out, tokens, choices, hidden, None)

    for name in ("y", "rows", "weights", "out"):
        assert combine(**{name: None}) == native.E_INVALID_ARGUMENT
    assert combine(tokens=-1) == native.E_UNSUPPORTED_SHAPE
    assert combine(choices=0) == native.E_UNSUPPORTED_SHAPE
    assert combine(hidden=12) == native.E_UNSUPPORTED_SHAPE
    assert combine(y=24) == native.E_MISALIGNED
    assert combine(rows=18) == native.E_MISALIGNED
    assert combine(tokens=0) == 0


def test_an_empty_gate_is_not_the_same_as_none(library):
    """The address of a gate of no rows is null, which stands for no gate: it is refused, not left out."""
    for gates in (0, 3):
        with pytest.raises(ValueError):
            int8.residual_norm(ones(4, 8), ones(4, 8), gate=ones(gates, 8), next_weight=ones(8))
    assert library.nvfp4_residual_norm(16, 0, 8, 16, 0, 8, None, None, 2, 1.0, 16, 1e-6, 16, 8, 16, 0, 8, None,
                                       4, 8, None) == native.E_INVALID_ARGUMENT


def test_norms_of_no_tokens_are_no_error(library):
    """The address of an empty tensor is null: without tokens a null residual stands for nothing, and what
    does not fit together is refused by the function for any number of tokens."""
    for post, gate, gates, scale in ((16, None, 0, 1.0), (None, 16, 1, 1.0), (None, None, 0, 0.5)):
        for weight in (16, None):
            assert library.nvfp4_residual_norm(None, 0, 8, None, 0, 8, post, gate, gates, scale, weight, 1e-6,
                                               None, 8, None, 0, 8, None, 0, 8, None) == 0
    w = ones(8)
    for wrong in (dict(post_weight=w), dict(gate=w), dict(residual_scale=0.5), dict(residual_out=ones(0, 8))):
        for tokens in (0, 4):
            with pytest.raises(ValueError):
                int8.residual_norm(ones(tokens, 8), next_weight=w, **wrong)


def test_an_eps_whose_root_has_no_fp32_reciprocal_is_refused(library):
    """1 / sqrt(eps) beyond FP32 would make NaN of a zero row."""
    def norm(eps):
        return library.nvfp4_residual_norm(None, 0, 8, None, 0, 8, None, None, 0, 1.0, 16, eps, None, 8, None, 0,
                                           8, None, 0, 8, None)

    for eps in (1e-77, 1e-6, 1e29):
        assert norm(eps) == 0
    for eps in (0.99e-77, 1e-100, 5e-324, 1e30, float("inf")):
        assert norm(eps) == native.E_INVALID_ARGUMENT


def test_functions_refuse_forward_gradients():
    """A tangent would be dropped without a word; operands without one pass the check inside a level of
    forward differentiation, under no_grad too (which does not switch it off)."""
    from torch.autograd import forward_ad

    a, b, sa, sb = codes(3, 32), codes(8, 32), ones(3), ones(8)
    experts, offsets = codes(2, 8, 32), torch.zeros(3, dtype=torch.int32)
    x, w = ones(4, 16), ones(16)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t.clone(), torch.ones_like(t))

        calls = (
            lambda: int8.gemm(a, b, dual(sa), sb),
            lambda: int8.gemm(a, b, sa, dual(sb)),
            lambda: int8.gemm(a, b, sa, sb, bias=dual(ones(8))),
            lambda: int8.gemm(a, b, sa, sb, out_dtype=torch.float32, out=dual(ones(3, 8))),
            lambda: int8.grouped_gemm(a, experts, dual(sa), ones(2, 8), offsets),
            lambda: int8.grouped_gemm(a, experts, sa, dual(ones(2, 8)), offsets),
            lambda: int8.quantize_tokens(dual(x)),
            lambda: int8.quantize_tokens(x, out=(codes(4, 16), dual(ones(4)))),
            lambda: int8.residual_norm(dual(x), next_weight=w),
            lambda: int8.residual_norm(x, dual(x), next_weight=w),
            lambda: int8.residual_norm(x, x, post_weight=dual(w), next_weight=w),
            lambda: int8.residual_norm(x, x, gate=dual(w), next_weight=w),
            lambda: int8.residual_norm(x, next_weight=dual(w)),
            lambda: int8.residual_norm(x, x, next_weight=w, residual_out=dual(x)),
            lambda: int8.residual_norm(x, next_weight=w, out=dual(x)),
            lambda: int8.residual_norm(x, next_weight=w, quantize=True, out=(codes(4, 16), dual(ones(4)))),
        )
        for call in calls:
            with pytest.raises(ValueError):
                call()
            with torch.no_grad(), pytest.raises(ValueError):
                call()
        for call in (lambda: int8.gemm(a, b, sa, sb), lambda: int8.quantize_tokens(x),
                     lambda: int8.residual_norm(x, x, next_weight=w)):
            with pytest.raises(RuntimeError):       # no device
                call()


def test_counts_beyond_the_kernels_32_bits_are_refused(library):
    """An index that runs a step past 2^31 - 1 would turn negative."""
    most, over = 1 << 30, (1 << 30) + 1

    def quantize(source=None, rows=4, tokens=4, k=8):
        return library.nvfp4_int8_quantize(16, 0, 1 << 31, source, rows, tokens, k, 16, 1 << 31, 16, None)

    for wrong in (dict(k=over), dict(k=(1 << 31) - 1), dict(rows=over, tokens=over), dict(source=16, rows=over),
                  dict(source=16, tokens=over)):
        assert quantize(**wrong) == native.E_UNSUPPORTED_SHAPE
    assert quantize(rows=0, tokens=0, k=most) == 0
    assert library.nvfp4_residual_norm(16, 0, 8, 16, 0, 8, None, None, 0, 1.0, 16, 1e-6, 16, 8, 16, 0, 8, None,
                                       over, 8, None) == native.E_UNSUPPORTED_SHAPE


def test_rings_of_products_let_loads_run_ahead(tmp_path):
    """Every tile the products are cut into keeps two stages, so that loads and MMAs do not take turns,
    unless its whole depth is one stage; with staging or without, and within a block's shared memory."""
    import subprocess

    header = native.LIBRARY_PATH.parents[1] / "csrc" / "int8_ring.h"
    source = tmp_path / "rings.cpp"
    source.write_text(f'#include "{header}"\n' + r"""
#include <cstdio>
#include <initializer_list>
int main() {
  for (int ctas = 1; ctas <= 2; ++ctas)
    for (int tokens = 32 * ctas; tokens <= 256; tokens += 32)
      for (int k : {1, 128, 129, 256, 257, 857, 1024, 131071})
        for (int experts : {1, 2, 32, 1024})
          for (int may = 0; may <= (k <= 1024); ++may) {
            const int sub = ctas == 1 || tokens <= 128 ? 2 : 1;
            const nvfp4::Int8Ring r = nvfp4::int8_ring(ctas, tokens, sub, k, experts, may);
            std::printf("%d %d %d %d %d %d %d %d %d\n", ctas, tokens, sub, k, experts, may, r.stages, r.staged, r.bytes);
          }
}
""")
    program = tmp_path / "rings"
    subprocess.run(["g++", "-std=c++17", "-o", str(program), str(source)], check=True)
    lines = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert len(lines) == 15 * 4 * (7 * 2 + 1)
    for line in lines:
        ctas, tokens, sub, k, experts, may, stages, staged, used = map(int, line.split())
        assert stages >= (1 if k <= 128 * sub else 2), line
        assert stages <= 12 and used <= 232448 - 5 * 1024 and (may or not staged), line
        stage = sub * 128 * (128 + tokens // ctas)
        warps = 4 * min(tokens // 32, 4)
        assert used == 1024 + stages * stage + 8 * (experts + 1) + staged * warps * 2048, line
