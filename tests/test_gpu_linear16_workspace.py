"""Calls of the 16-bit Linear layer with exactly the workspace that they ask for, in a buffer whose rest stays as it
was, have the bits of calls with more; those that run in one launch take none."""
import pytest

from tests.gpu_util import require_gpu, say
from tests.test_gpu_linear16 import _act_code, _rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


@pytest.mark.parametrize("size", [(48, 200, 4096), (64, 8192, 4096), (8192, 256, 784), (16, 640, 6575), (300, 263, 1777),
                                  (700, 1032, 520), (130, 24, 0)])
@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
def test_exact_workspaces(size, act):
    import torch
    from cudeep_amd import _lib as L, ops
    M, N, K = size
    say("workspace", size, act)
    code = _act_code(act)
    x, w, b, dy, z = (_rnd((M, K), 1, "bf16"), _rnd((N, K), 2, "bf16"), _rnd((N,), 3, "bf16"), _rnd((M, N), 4, "bf16"),
                      _rnd((M, N), 5, "bf16"))
    lib = L.lib()

    def within(need, f, want):
        buf = torch.full((need // 16 * 16 + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
        got = f(buf[:max(need, 16)] if need else buf[:16])
        for a, c in zip(got, want):
            assert (a is None) == (c is None) and (a is None or torch.equal(a, c))
        assert (buf[need:] == 0x5A).all()

    need = lib.cdx_linear16_call_workspace_size(M, N, K, x.data_ptr(), K, w.data_ptr(), K)
    assert need <= ops.linear16_workspace_bytes(M, N, K)
    if K:
        within(need, lambda ws: (ops.linear16(x, w, b, epilogue=code, workspace=ws),), (ops.linear16(x, w, b, epilogue=code),))
    for input, params, bias in ((True, True, True), (True, False, False), (False, True, True), (False, True, False)):
        need = lib.cdx_linear16_backward_call_workspace_size(M, N, K, dy.data_ptr(), N, x.data_ptr(), K, w.data_ptr(), K, code,
                                                             input, params, bias)
        kw = dict(epilogue=code, input=input, params=params, bias=bias)
        within(need, lambda ws: ops.linear16_backward(dy, x, w, z, workspace=ws, **kw), ops.linear16_backward(dy, x, w, z, **kw))
