"""Layer norm's and the 8-bit operators' C entry points refuse bad arguments before any launch, and
their size queries answer without a GPU; the host restatement of the 8-bit format agrees with
torch's conversion."""
import ctypes

import numpy as np
import pytest

from cudeep_amd import _lib as L
from tests import block8_ref as ref

P = ctypes.c_void_p(0x1000)   # never dereferenced: validation fails first
F32, F64, F16, BF16, E8 = 0, 1, 2, 3, 4


def _status(name, *args):
    return getattr(L.lib(), name)(*args)


def _bad(name, good, changes):
    """Every change {position: value} of the good arguments is refused."""
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert _status(name, *args) == L.CDX_ERR_INVALID_ARG, (name, at, value)
        assert name.encode() in L.lib().cdx_last_error()


def test_layer_norm_arguments():
    good = [P, 8, P, P, P, 8, P, P, 4, 8, 1e-5, F32, F32, None]
    _bad("cdx_layer_norm_forward", good, [
        (0, None), (1, 7), (4, None), (5, 7), (8, -1), (9, 0), (9, -1), (10, -1.0),
        (10, float("nan")), (10, float("inf")), (11, F64), (11, 9), (12, F16)])
    assert _status("cdx_layer_norm_forward", None, 8, None, None, None, 8, None, None, 0, 8, 1e-5,
                   F32, F32, None) == L.CDX_OK
    good = [P, 8, P, 8, P, P, P, P, 8, P, P, 4, 8, F32, F32, P, 1 << 20, None]
    _bad("cdx_layer_norm_backward", good, [
        (0, None), (1, 7), (2, None), (3, 7), (5, None), (6, None), (7, None), (8, 7), (11, -1),
        (12, 0), (13, F64), (14, BF16)])
    small = list(good)
    small[16] = 4
    assert _status("cdx_layer_norm_backward", *small) == L.CDX_ERR_WORKSPACE
    assert _status("cdx_layer_norm_backward_workspace_size", 4, 8, F32) >= 2 * 8 * 4
    assert _status("cdx_layer_norm_backward_workspace_size", 0, 8, F32) == 0


def test_quantizer_arguments():
    good = [P, 200, 40, 200, F32, 1, P, 200, P, 2, E8, None]
    _bad("cdx_quantize_e4m3", good, [
        (0, None), (1, 199), (2, -1), (3, -1), (4, F64), (5, 2), (5, 0), (6, None), (7, 199),
        (8, None), (9, 1), (10, F16)])
    assert _status("cdx_quantize_e4m3", None, 200, 0, 200, F32, 1, None, 200, None, 2, E8, None) == L.CDX_OK
    good = [P, 200, P, 2, E8, 1, P, 200, 40, 200, F32, None]
    _bad("cdx_dequantize_e4m3", good, [
        (0, None), (1, 199), (2, None), (3, 1), (4, BF16), (5, 3), (6, None), (7, 199), (8, -1),
        (10, F64)])


def test_product_arguments():
    good = [4, 8, 200, P, 200, P, 2, E8, P, 200, P, 2, E8, P, 8, BF16, None, 0, None, 0, None]
    _bad("cdx_gemm_e4m3", good, [
        (0, -1), (1, -1), (2, -1), (3, None), (4, 199), (5, None), (6, 1), (7, F16), (8, None),
        (9, 199), (10, None), (11, 1), (12, F16), (13, None), (14, 7), (15, F64), (17, 5), (17, 9)])
    good = [4, 8, 200, P, 200, BF16, P, 200, P, 2, E8, P, 8, BF16, None, 0, P, 1 << 20, None]
    _bad("cdx_linear_e4m3", good, [
        (0, -1), (3, None), (4, 199), (5, F64), (6, None), (7, 199), (8, None), (9, 1), (10, F16),
        (11, None), (12, 7), (13, F64), (15, 5)])
    small = list(good)
    small[0] = 400
    small[17] = 4
    assert _status("cdx_linear_e4m3", *small) == L.CDX_ERR_WORKSPACE
    assert _status("cdx_linear_e4m3_workspace_size", 400, 8, 200) >= 400 * 200
    assert _status("cdx_gemm_e4m3", 0, 8, 200, None, 200, None, 2, E8, P, 200, P, 2, E8, None, 8, BF16,
                   None, 0, None, 0, None) == L.CDX_OK


def test_checkpoint_arguments():
    good = [P, 200, P, 200, P, 200, P, 2, E8, 40, 200, F32, 2, 0.0, None]
    _bad("cdx_activation_forward_e4m3", good, [
        (0, None), (1, 199), (2, None), (3, 199), (4, None), (5, 199), (6, None), (7, 1), (8, F16),
        (9, -1), (11, F64), (12, 0), (12, 7), (12, 9)])
    good = [P, 200, P, 200, P, 2, E8, P, 200, 40, 200, F32, 2, 0.0, None]
    _bad("cdx_activation_backward_e4m3", good, [
        (0, None), (1, 199), (2, None), (3, 199), (4, None), (5, 1), (6, F16), (7, None), (8, 199),
        (9, -1), (11, F64), (12, 0)])
    good = [P, 8, F32, P, 200, P, 2, P, P, 40, 8, 200, P, 1 << 30, None]
    _bad("cdx_linear_weight_grad_e4m3", good, [
        (0, None), (1, 7), (2, F64), (3, None), (4, 199), (5, None), (6, 1), (7, None), (9, -1),
        (10, -1), (11, -1)])
    many = list(good)
    many[9] = 1 << 14
    many[13] = 4
    assert _status("cdx_linear_weight_grad_e4m3", *many) == L.CDX_ERR_WORKSPACE
    assert _status("cdx_linear_weight_grad_e4m3_workspace_size", 1 << 14, 8, 200, F32) > 8 * 200 * 4


def test_host_format_agrees_with_torch():
    torch = pytest.importorskip("torch")
    codes = np.arange(256, dtype=np.uint8)
    v = torch.from_numpy(codes).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(np.isnan(v), np.isnan(ref.CODES))
    assert np.array_equal(v[~np.isnan(v)], ref.CODES[~np.isnan(v)].astype(np.float32))
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.uniform(-448, 448, 4000), rng.standard_normal(4000) * 0.02,
                        (ref._POS[1:] + ref._POS[:-1]) / 2]).astype(np.float32)   # ties too
    t = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref.round_codes(x), t)


def test_wrappers_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    from cudeep_amd import ops
    x = torch.zeros(4, 8)
    b = ops.Block8(x.to(torch.float8_e4m3fn), torch.ones(4, 1), 1)
    for f in (lambda: ops.layer_norm(x), lambda: ops.quantize8(x), lambda: ops.dequantize8(b),
              lambda: ops.gemm8(b, b), lambda: ops.linear8(x, b), lambda: ops.activation8(x, 1),
              lambda: ops.activation_backward8(x, b, 1), lambda: ops.linear_weight_grad8(x, b)):
        with pytest.raises((ValueError, TypeError)):
            f()
