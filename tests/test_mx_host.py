"""Microscaled operators without a GPU: the C ABI's table and refusals, shapes and refusals of the operators, the module, and
the oracle against the formats' own numbers."""
import ctypes
import os
import re

import pytest
import torch

import nanoquantization_amd as nq
from nanoquantization_amd import _lib
from oracle import mx_oracle as mx

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FORMATS = ("mxfp4", "mxfp8")


@pytest.fixture(scope="module", autouse=True)
def built():
    if not (os.path.exists(_lib.MX_LIB_PATH) and os.path.exists(_lib.MX_TORCH_LIB_PATH)):
        from nanoquantization_amd.build import build_mx
        build_mx(verbose=False)


def test_header_and_ctypes_table_agree():
    header = open(os.path.join(ROOT, "include", "nq_mx_ops.h")).read()
    header = re.sub(r"/\*.*?\*/", "", header, flags=re.S)
    declared = set(re.findall(r"\b(nqx_\w+)\s*\(", header))
    assert declared == set(_lib.MX_SYMBOLS)
    handle = ctypes.CDLL(_lib.MX_LIB_PATH)
    for name in declared:
        assert hasattr(handle, name)


def test_c_abi_refuses_before_it_launches():
    L = _lib.mx_lib()
    at = 4096                                                # never read: every call below is refused
    sizes = dict(rows=4, n=64, k=64)

    def quantize(x=at, stride=64, codes=at, scales=at, rows=4, k=64, dtype=1, fmt=0):
        return L.nqx_quantize(x, stride, codes, scales, rows, k, dtype, fmt, None)

    assert quantize(dtype=3) == quantize(dtype=-1) == 1
    assert quantize(fmt=2) == 1 and b"format" in L.nqx_last_error()
    assert quantize(k=48) == 1 and b"multiple of 32" in L.nqx_last_error()
    assert quantize(k=0) == quantize(rows=-1) == 1
    assert quantize(x=None) == quantize(x=at + 8) == quantize(codes=at + 4) == quantize(scales=None) == 1
    assert quantize(stride=63) == quantize(stride=-64) == 1 and b"16-byte" in L.nqx_last_error()
    assert quantize(rows=1 << 33) == 2
    assert quantize(rows=0, x=None, codes=None, scales=None) == 0

    def dequantize(codes=at, scales=at, y=at, rows=4, k=64, dtype=1, fmt=0):
        return L.nqx_dequantize(codes, scales, y, rows, k, dtype, fmt, None)

    assert dequantize(codes=None) == dequantize(codes=at + 1) == dequantize(scales=None) == dequantize(y=at + 2) == 1
    assert dequantize(rows=0, y=None) == 0

    def product(codes=at, scales=at, w=at, ws=at, y=at, rows=4, n=64, k=64, dtype=1, fmt=1):
        return L.nqx_linear_quantized(codes, scales, w, ws, None, y, rows, n, k, dtype, fmt, at, 1 << 30, None)

    assert product(codes=None) == product(codes=at + 8) == product(scales=None) == product(w=at + 8) == product(ws=None) == 1
    assert product(y=None) == product(n=-1) == product(k=40) == 1
    assert product(rows=(1 << 20) + 1) == product(n=(1 << 30) + 1) == 2
    assert product(rows=0, codes=None) == product(n=0, w=None) == 0

    def linear(x=at, stride=64, ws_bytes=1 << 20, space=at, rows=64, dtype=1, fmt=1):
        # 64 rows: quantised in front of the product
        return L.nqx_linear(x, stride, at, at, None, at, rows, 64, 64, dtype, fmt, space, ws_bytes, None)

    need = L.nqx_linear_workspace_bytes(64, 64, 64, 1, 1, 0)
    assert need >= 64 * 64 + 64 * 2
    assert linear(ws_bytes=need - 1) == linear(space=None) == linear(space=at + 8) == 3 and b"workspace" in L.nqx_last_error()
    assert linear(x=at + 2) == linear(stride=60) == linear(dtype=5) == linear(fmt=-1) == 1
    assert L.nqx_linear_workspace_bytes(64, 64, 33, 1, 1, 0) == 0
    # a product whose k is split over workgroups has sums to keep
    split = L.nqx_linear_workspace_bytes(20, 256, 8192, 1, 1, 1)
    assert split >= 20 * 256 * 4 * 2
    assert L.nqx_linear_quantized(at, at, at, at, None, at, 20, 256, 8192, 1, 1, at, split - 1, None) == 3
    assert L.nqx_linear_quantized(at, at, at, at, None, at, 20, 256, 8192, 1, 1, None, split, None) == 3

    def norm(x=at, xs=64, delta=at, ds=64, weight=at, total=at, codes=at, scales=at, rows=4, k=64, dtype=1, fmt=1):
        return L.nqx_add_rmsnorm(x, xs, delta, ds, weight, total, codes, scales, rows, k, 1e-6, dtype, fmt, None)

    assert norm(k=16384 + 32) == 2 and b"16384" in L.nqx_last_error()
    assert norm(weight=None) == norm(total=None) == norm(x=None) == norm(delta=at + 2) == norm(codes=None) == 1
    assert norm(xs=128) == 1 and b"k apart" in L.nqx_last_error()      # total is x, whose rows are not dense
    assert norm(x=2 * at, ds=128) == 1
    assert norm(rows=0) == 0

    def silu(gate=at, gs=64, up=at, us=64, codes=at, scales=at, rows=4, k=64, dtype=1, fmt=1):
        return L.nqx_silu_mul(gate, gs, up, us, codes, scales, rows, k, dtype, fmt, None)

    assert silu(gate=None) == silu(up=at + 4) == silu(gs=60) == silu(us=1) == silu(codes=None) == silu(k=31) == 1
    assert silu(rows=0) == 0
    assert L.nqx_linear_form(*sizes.values(), 1, 1, 1) != b"" and L.nqx_linear_form(4, 64, 33, 1, 1, 1) == b""


def _meta(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device="meta")


def test_meta_shapes():
    ops = _lib.mx_ops()
    for fmt, per in (("mxfp4", 2), ("mxfp8", 1)):
        codes, scales = ops.mx_quantize(_meta(3, 5, 96), fmt)
        assert codes.shape == (3, 5, 96 // per) and scales.shape == (3, 5, 3) and codes.dtype == scales.dtype == torch.uint8
        assert ops.mx_dequantize(codes, scales, torch.float32).shape == (3, 5, 96)
        w, ws = _meta(7, 48, dtype=torch.uint8), _meta(7, 3, dtype=torch.uint8)
        y = ops.mx_linear_quantized(codes, scales, w, ws, None, torch.float16)
        assert y.shape == (3, 5, 7) and y.dtype == torch.float16
        assert ops.mx_linear(_meta(96), w, ws, None, fmt).shape == (7,)
        c, s, total = ops.mx_add_rmsnorm(_meta(4, 96), _meta(4, 96), _meta(96), 1e-6, fmt)
        assert c.shape == (4, 96 // per) and s.shape == (4, 3) and total.shape == (4, 96) and total.dtype == torch.bfloat16
        assert ops.mx_silu_mul(_meta(4, 96), _meta(4, 96), fmt)[0].shape == (4, 96 // per)
    assert ops.mx_quantize(_meta(0, 64), "mxfp8")[0].shape == (0, 64)


def test_operators_refuse():
    ops = _lib.mx_ops()
    w, ws = _meta(7, 48, dtype=torch.uint8), _meta(7, 3, dtype=torch.uint8)
    x, c8, s = _meta(4, 96), _meta(4, 96, dtype=torch.uint8), _meta(4, 3, dtype=torch.uint8)
    for call in (lambda: ops.mx_quantize(x, "mxfp6"), lambda: ops.mx_quantize(_meta(4, 40), "mxfp4"),
                 lambda: ops.mx_quantize(_meta(4, 64, dtype=torch.float64), "mxfp4"), lambda: ops.mx_quantize(_meta(), "mxfp4"),
                 lambda: ops.mx_dequantize(c8, s[:3], torch.float32), lambda: ops.mx_dequantize(c8[:, :64], s, torch.float32),
                 lambda: ops.mx_dequantize(c8.to(torch.int8), s, torch.float32), lambda: ops.mx_dequantize(c8, s, torch.float64),
                 lambda: ops.mx_linear(x, _meta(7, 96, dtype=torch.uint8), ws, None, "mxfp8"),       # the weight is not mxfp4
                 lambda: ops.mx_linear(_meta(4, 64), w, ws, None, "mxfp8"), lambda: ops.mx_linear(x, w, ws, None, "fp8"),
                 lambda: ops.mx_linear_quantized(c8, s, w, ws[:, :2], None, torch.float16),
                 lambda: ops.mx_add_rmsnorm(x, _meta(5, 96), _meta(96), 1e-6, "mxfp8"),
                 lambda: ops.mx_add_rmsnorm(x, x, _meta(64), 1e-6, "mxfp8"),
                 lambda: ops.mx_add_rmsnorm(x, x, _meta(96, dtype=torch.float32), 1e-6, "mxfp8"),
                 lambda: ops.mx_rmsnorm(_meta(1, 16416), _meta(16416), 1e-6, "mxfp8"),
                 lambda: ops.mx_silu_mul(x, _meta(4, 96, dtype=torch.float16), "mxfp8")):
        with pytest.raises(RuntimeError):
            call()


def test_host_tensors_are_refused():
    x, w, ws = torch.zeros(2, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8)
    for call in (lambda: nq.mx_quantize(x), lambda: nq.mx_dequantize(w, ws), lambda: nq.mx_linear(x, w, ws),
                 lambda: nq.mx_linear_quantized(w, ws, w, ws), lambda: nq.mx_add_rmsnorm(x, x, x[0]),
                 lambda: nq.mx_add_rmsnorm(x, None, x[0]), lambda: nq.mx_silu_mul(x, x),
                 lambda: nq.MXLinear(64, 8)(x), lambda: nq.MXLinear.from_linear(torch.nn.Linear(64, 8))):
        with pytest.raises(_lib.AwqHipError):
            call()
    with pytest.raises(NotImplementedError):      # no CPU kernel is registered: there is no fallback to fall into
        _lib.mx_ops().mx_quantize(x, "mxfp4")


def test_module_buffers():
    m = nq.MXLinear(96, 40, bias=True)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {"weight": (40, 48), "weight_scales": (40, 3), "bias": (40,)}
    assert m.bias.dtype == torch.bfloat16 and nq.MXLinear(64, 8).bias is None
    with pytest.raises(ValueError):
        nq.MXLinear(64, 8, activations="mxfp6")
    with pytest.raises(AssertionError):
        nq.MXLinear(48, 8)


def test_oracle_elements():
    assert mx.elements("mxfp4").tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    e8 = mx.elements("mxfp8")
    assert e8[-1] == 448 and e8[1] == 2.0 ** -9 and e8[8] == 2.0 ** -6
    codes = torch.arange(127, dtype=torch.uint8)
    assert torch.equal(codes.view(torch.float8_e4m3fn).double(), e8)


@pytest.mark.parametrize("fmt", FORMATS)
def test_oracle_rounds_by_half_a_step_at_most(fmt):
    torch.manual_seed(0)
    x = torch.randn(64, 128, dtype=torch.float64) * torch.logspace(-30, 30, 64, dtype=torch.float64).unsqueeze(1)
    codes, scales = mx.quantize(x, fmt)
    assert ((mx.values(codes, scales) - x).abs() <= mx.half_steps(x, scales.to(torch.int64) - 127, fmt)).all()
    again, s = mx.quantize(mx.values(codes, scales), fmt)
    # values that are elements already stay what they are
    assert torch.equal(mx.values(again, s), mx.values(codes, scales))


def test_oracle_scales():
    def byte(v, fmt):
        return int(mx.quantize(torch.tensor([v] + [0.0] * 31, dtype=torch.float64), fmt)[1])
    below = 7.0 - 2.0 ** -30
    assert byte(6.0, "mxfp4") == byte(below, "mxfp4") == 127 and byte(7.0, "mxfp4") == 128 and byte(4.0, "mxfp4") == 127
    assert byte(448.0, "mxfp8") == byte(464.0, "mxfp8") == 127 and byte(464.0 + 2.0 ** -30, "mxfp8") == 128
    assert byte(0.0, "mxfp4") == byte(2.0 ** -149, "mxfp8") == 0
    assert byte(float("inf"), "mxfp4") == byte(float("nan"), "mxfp8") == 255


def test_sizes_past_a_launch_are_refused():
    """2^36 values and more, 2^24 rows of a norm, weights of more than 2^29 rows: refused before a pointer is looked at."""
    L, at = _lib.mx_lib(), 4096
    assert L.nqx_quantize(at, 1 << 16, at, at, 1 << 20, 1 << 16, 1, 0, None) == 2 and b"too large" in L.nqx_last_error()
    assert L.nqx_dequantize(at, at, at, 1 << 31, 32, 1, 0, None) == 2
    assert L.nqx_silu_mul(at, 1 << 16, at, 1 << 16, at, at, 1 << 20, 1 << 16, 1, 0, None) == 2
    assert L.nqx_add_rmsnorm(at, 32, None, 0, at, None, at, at, 1 << 24, 32, 1e-6, 1, 0, None) == 2 and b"2^24" in L.nqx_last_error()
    assert L.nqx_linear_workspace_bytes(1, (1 << 29) + 1, 32, 1, 0, 0) == 0
    assert L.nqx_linear(at, 32, at, at, None, at, 1, (1 << 29) + 1, 32, 1, 0, None, 0, None) == 2


def test_largest_sizes_of_a_launch():
    """The last sizes below 2^36 values, whose last workgroup would be past 2^32 threads, are refused by name, not by the launch."""
    L, at = _lib.mx_lib(), 4096
    for rows, k in (((1 << 31) - 1, 32), ((1 << 31) - 127, 32), (((1 << 31) - 1) // 3, 96)):
        assert L.nqx_silu_mul(at, k, at, k, at, at, rows, k, 1, 0, None) == 2 and b"too large" in L.nqx_last_error()
        assert L.nqx_quantize(at, k, at, at, rows, k, 1, 0, None) == 2 and L.nqx_dequantize(at, at, at, rows, k, 1, 0, None) == 2


def test_meta_kernels_check_what_device_kernels_check():
    """A bias of another size or rank, and tensors of two devices, pass neither tracing nor the device."""
    ops = _lib.mx_ops()
    w, ws, x = _meta(7, 48, dtype=torch.uint8), _meta(7, 3, dtype=torch.uint8), _meta(4, 96)
    c8, s = _meta(4, 96, dtype=torch.uint8), _meta(4, 3, dtype=torch.uint8)
    for good in (None, _meta(7), _meta(7, dtype=torch.float32), _meta(7, dtype=torch.float16)):
        assert ops.mx_linear(x, w, ws, good, "mxfp8").shape == ops.mx_linear_quantized(c8, s, w, ws, good, torch.float16).shape == (4, 7)
    for bad in (_meta(8), _meta(1), _meta(7, 1), _meta(0), torch.zeros(7, dtype=torch.bfloat16)):
        for call in (lambda: ops.mx_linear(x, w, ws, bad, "mxfp8"), lambda: ops.mx_linear_quantized(c8, s, w, ws, bad, torch.float16)):
            with pytest.raises(RuntimeError):
                call()
    cpu, cpu8 = torch.zeros(4, 96, dtype=torch.bfloat16), torch.zeros(4, 3, dtype=torch.uint8)
    for call in (lambda: ops.mx_linear(x, torch.zeros(7, 48, dtype=torch.uint8), ws, None, "mxfp8"), lambda: ops.mx_dequantize(c8, cpu8, torch.float16),
                 lambda: ops.mx_linear_quantized(c8, cpu8, w, ws, None, torch.float16), lambda: ops.mx_silu_mul(x, cpu, "mxfp8"),
                 lambda: ops.mx_add_rmsnorm(x, cpu, _meta(96), 1e-6, "mxfp8"), lambda: ops.mx_rmsnorm(x, cpu[0], 1e-6, "mxfp8")):
        with pytest.raises(RuntimeError):
            call()
