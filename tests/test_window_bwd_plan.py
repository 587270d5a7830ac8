'''The windowed backward's workspace with many first tokens, read from the size it asks for (no GPU): the
partial sums behind the windows are cut into chunks to fill the chip, not to fill memory.'''
import pytest

from motif.ops import _lib

MB = 1 << 20


def _bytes(B, H, Hkv, L, S, q_start, window, sinks):
    return _lib.lib().motif_chord_window_bwd_workspace_bytes(B, H, Hkv, L, S, q_start, window, sinks)


def _without_chunks(B, H, Hkv, L, S, window):
    '''What the same call takes with no first tokens: row values, parameter sums, and (shared heads) the keys'
    own partials.'''
    return _bytes(B, H, Hkv, L, S, S - L, window, 0)


@pytest.mark.parametrize('B,H,Hkv,S', [(1, 12, 3, 8192), (1, 12, 12, 8192), (8, 12, 3, 8192), (2, 16, 4, 65536), (64, 12, 3, 2048),
                                       (1, 1, 1, 262144)])
def test_chunks_stop_where_the_chip_is_full(B, H, Hkv, S):
    '''Two fp32 rows of 64 features per head and key for each chunk: as many chunks as eight workgroups per CU
    ask for (2048 of 128 rows: 134 MB), or one.'''
    plane = 2 * 64 * 4 * B * H * S
    for sinks in (S - 1, S // 2, S // 16):
        extra = _bytes(B, H, Hkv, S, S, 0, 64, sinks) - _without_chunks(B, H, Hkv, S, S, 64)
        if H == Hkv:  # (the blocks of first tokens have partials of their own windows)
            extra -= 2 * 64 * 4 * B * H * -(-sinks // 128) * 128
        assert extra <= max(2048 * 128 * 512, plane) + MB, (sinks, extra / MB)


@pytest.mark.parametrize('sinks', [1, 4, 128, 1000])
def test_few_first_tokens_keep_their_chunks(sinks):
    '''16 chunks of 8192 queries behind a window of 64 while they are fewer than 2048 workgroups.'''
    B, H, Hkv, S = 1, 12, 3, 8192
    blocks = -(-sinks // 128)
    extra = _bytes(B, H, Hkv, S, S, 0, 64, sinks) - _without_chunks(B, H, Hkv, S, S, 64)
    chunks = extra / (2 * 64 * 4 * B * H * blocks * 128)
    assert 15 <= chunks <= 16.1
