"""How the sequence operators cut their work up, from the buffer sizes that the C entries report (no GPU needed): tests that mean to reach a loop's
second turn check here that they do."""
import ctypes as C

from gan_amd import _lib as L


def scan_plan(B, T, Cn, N, G):
    """(chunks of a sequence, tiles of 16 rows in a chunk)"""
    s = L.ScanBuffers()
    assert L.lib().ga_scan_sizes(B, T, Cn, N, G, C.byref(s)) == 0
    padded = next(n for n in (8, 16, 32, 64) if N <= n)
    chunks, rest = divmod(s.dparams, B * (padded + 2) * Cn)
    assert rest == 0
    tiles = -(-T // 16)
    return chunks, -(-tiles // chunks)


def conv_bwd_plan(B, T, Cn, K):
    """(blocks along time of the backward pass at the most, the fewest turns of its loop over runs).  Runs are 128 rows at the most; a block takes four
    of them at a time where a row has 33 channel pieces or more, else up to 256."""
    parts = L.lib().ga_causal_conv_bwd_ws_elems(B, T, Cn, K) // ((K + 1) * Cn)
    pieces = Cn // (4 if K <= 4 else 2) if Cn % 4 == 0 else Cn
    at_once = 4 if pieces > 32 else 256
    return parts, -(-(B * -(-T // 128)) // (parts * at_once))


def norm_plan(B, T, Cn, by_item, vec):
    """(rows of an item, the fewest turns of the loops over rows in the forward and the backward pass): rows a block works on at a time, by width"""
    items = B if by_item else 1
    rows = T if by_item else B * T
    parts = (L.lib().ga_block_norm_bwd_ws_elems(B, T, Cn, int(by_item)) // (4 * Cn) - (items if by_item else 0)) // items
    if vec:
        fwd, bwd = (16, 8) if Cn <= 256 else (8, 4) if Cn <= 512 else (4, 2) if Cn <= 1024 else (2, 1) if Cn <= 2048 else (1, 1)
    else:
        fwd, bwd = (8, 4) if Cn <= 256 else (2, 1) if Cn <= 1024 else (1, 1)
    return rows, -(-rows // (parts * fwd)), -(-rows // (parts * bwd))
