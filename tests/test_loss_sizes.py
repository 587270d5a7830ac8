'''How large the arguments of linear_cross_entropy's C entries may be (host only): what a launch cannot hold is refused, in the
forward as in the backward, and has no workspace.'''
import ctypes

import pytest

from motif.ops import _lib

P = ctypes.c_void_p(16)  # (never read: every call below ends at a check)


def _entries(N, d, V, dtype):
    lib = _lib.lib()
    fwd = lib.motif_linear_ce_fwd(P, d, P, d, P, 1, -100, N, d, V, 2, P, P, P, P, 0, dtype, None)
    said = lib.motif_last_error().decode()
    bwd = lib.motif_linear_ce_bwd(P, P, d, P, P, 1, N, d, V, 2, P, P, P, 0, dtype, None)
    return fwd, bwd, said, lib.motif_last_error().decode(), [lib.motif_linear_ce_workspace_bytes(N, d, P, d, V, dtype, b) for b in (0, 1)]


@pytest.mark.parametrize('N,d,V,dtype', [
    (2 ** 23, 2 ** 16, 1, 1), (2 ** 23, 2 ** 15 + 2 ** 14, 2 ** 22 - 64, 1), (2 ** 23, 2 ** 14, 1, 0), (2 ** 20, 2 ** 16, 1, 0), (1, 2 ** 16, 2 ** 20, 0),
])
def test_more_than_a_launch_holds(N, d, V, dtype):
    fwd, bwd, said_fwd, said_bwd, space = _entries(N, d, V, dtype)
    assert fwd == bwd == _lib.ERR_INVALID and 'out of range' in said_fwd and 'out of range' in said_bwd and space == [0, 0]


@pytest.mark.parametrize('N,d,V,dtype', [
    (2 ** 23, 513, 2, 1), (2 ** 22 + 128, 8, 2 ** 17, 1), (2 ** 23, 1024, 2 ** 17, 1), (2 ** 20, 1024, 2 ** 17, 0), (2 ** 10, 2 ** 16, 2 ** 17, 0),
])
def test_what_it_holds(N, d, V, dtype):
    fwd, bwd, said_fwd, said_bwd, space = _entries(N, d, V, dtype)  # (refused for the workspace alone)
    assert fwd == bwd == _lib.ERR_INVALID and 'workspace' in said_fwd and 'workspace' in said_bwd
    # a forward has two numbers for each row and 128 (bf16) or 32 (fp32) words, a backward P of 256 words and dX once
    words = 128 if dtype else 32
    assert space[0] >= 8 * N * (V // words) and space[1] >= N * 256 * (2 if dtype else 4) + 4 * N * d


def test_norm_workgroups():
    '''A partial row for each of at most 512 workgroups, twice for LayerNorm.'''
    need = _lib.lib().motif_row_norm_bwd_workspace_bytes
    assert need(511, 64, 0) == 511 * 64 * 4 and need(10 ** 6, 64, 0) == 512 * 64 * 4 and need(2 ** 31 - 1, 16384, 1) == 2 * 512 * 16384 * 4
