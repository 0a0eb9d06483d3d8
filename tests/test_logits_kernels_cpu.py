"""The library holds the kernels that a call can reach, and no others of the same families (no GPU needed: names of
kernels as they are registered)."""
import re

from cudeep_amd import _lib as L


def _kernels(name):
    """Template arguments, as mangled, of a family's kernels."""
    data = open(L.LIB_PATH, "rb").read()
    return set(re.findall(rb"\d+%sI(\w+?)EEv" % name, data))


def test_threads_of_log_probabilities():
    found = _kernels(b"logprob_kernel")
    for threads in (256, 512, 1024):
        for dtype in (b"f", b"DF16_", b"DF16b"):
            for entropy in (b"0", b"1"):
                for top in (b"0", b"1"):
                    name = dtype + b"Li%dELb" % threads + entropy + b"ELb" + top + b"E"
                    assert (name in found) == (threads < 1024 or top == b"0"), name


def test_activations_of_the_slopes():
    """ReLU (1), GELU (2), SiLU (3), sigmoid (4); with sums, those that round."""
    for family, acts in ((b"linear16_slope_kernel", b"1234"), (b"linear16_slope_sums_kernel", b"234")):
        assert {f[re.search(rb"Li(\d)", f).start(1):][:1] for f in _kernels(family)} == {bytes([a]) for a in acts}
