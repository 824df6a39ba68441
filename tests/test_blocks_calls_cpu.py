"""What the layer operators' host side answers without a GPU, beside test_blocks_cpu.py: workspaces and refusals at the edges of the sizes."""
import ctypes as C

from isbfsar_amd import _lib
from test_blocks_cpu import lib, norm, xattn                                       # noqa: F401  (the fixture)


def test_norm_workspace_does_not_grow_with_the_samples(lib):                  # noqa: F811
    """short samples with a gate: partial sums per workgroup, not per sample"""
    n = C.c_size_t()
    for B, L, D in ((65535, 1, 8192), (65535, 2, 8192), (65535, 16, 2048), (65535, 1, 64), (4000, 2, 512), (300, 1, 8192), (1, 1 << 20, 8192)):
        assert lib.isb_norm_workspace(C.byref(norm(B=B, L=L, D=D, gate=4096)), C.byref(n)) == 0
        assert 0 < n.value <= 160 << 20, (B, L, D, n.value)


def test_xattn_workgroups_are_rounded_up_to_the_xcds(lib):                    # noqa: F811
    """2^23 workgroups of 512 threads are 2^32: one more than a launch holds"""
    n = C.c_size_t()
    one = dict(Lq=1, Lk=1, Hq=1, Hk=1, D=8, strides=(8, 8, 8))
    for tiles, rc in (((1 << 23) - 8, 0), ((1 << 23) - 7, -1), ((1 << 23) - 1, -1), (1 << 23, -1)):
        a = xattn(B=tiles, Bk=tiles, **one)
        assert lib.isb_xattn_workspace(C.byref(a), 0, C.byref(n)) == rc, tiles
        assert rc == 0 or lib.isb_xattn_forward(C.byref(a), 4096, 1 << 40, None) == -1
