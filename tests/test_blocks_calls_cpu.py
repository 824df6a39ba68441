"""What the layer operators' host side answers without a GPU, beside test_blocks_cpu.py: workspaces and refusals at the edges of the sizes."""
import ctypes as C

from isbfsar_amd import _lib
from test_blocks_cpu import lib, norm                                         # noqa: F401  (the fixture)


def test_norm_workspace_does_not_grow_with_the_samples(lib):                  # noqa: F811
    """short samples with a gate: partial sums per workgroup, not per sample"""
    n = C.c_size_t()
    for B, L, D in ((65535, 1, 8192), (65535, 2, 8192), (65535, 16, 2048), (65535, 1, 64), (4000, 2, 512), (300, 1, 8192), (1, 1 << 20, 8192)):
        assert lib.isb_norm_workspace(C.byref(norm(B=B, L=L, D=D, gate=4096)), C.byref(n)) == 0
        assert 0 < n.value <= 160 << 20, (B, L, D, n.value)
