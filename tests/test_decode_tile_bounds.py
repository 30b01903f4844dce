"""CPU: the rows of a tile that the decode kernel clears, restated from its source, when a sequence's length changes between the
kernel's reads of it (a caller that rewrites ``seq_lens`` without waiting for the launch).  The result is then nobody's, but no
row outside the tile may be written: shared memory of other warps lies there, and further out nothing."""
from pathlib import Path

SOURCE = (Path(__file__).resolve().parents[1] / "nanopd_b200" / "csrc" / "decode_kernel.cuh").read_text()
TILE = 16


def test_the_source_is_what_is_restated_here():
    assert "const int valid = max(0, min(kTile, seg_len - tok0));" in SOURCE
    assert "const int cnt = min(seg_lo - tok0, kTile) * NH * 8;" in SOURCE
    assert "boxes = max(0, min(kTile, pc.len - tok0 + p.box_rows - 1)) >> p.box_shift;" in SOURCE


def test_rows_cleared_and_boxes_requested_stay_in_the_tile():
    for first_read in (1, 15, 16, 17, 300, 17000):
        for second_read in (0, 1, 16, 299, 12000, 17008):
            for window in (1, 16, 40, 1 << 30):
                first = lambda n: max(0, n - window) // TILE  # noqa: E731
                for t in range((first_read + TILE - 1) // TILE - first(first_read)):
                    tok0 = (first(second_read) + t) * TILE
                    valid = max(0, min(TILE, second_read - tok0))
                    assert 0 <= valid <= TILE                           # rows valid .. 15 behind the sequence are cleared
                    lo = max(0, second_read - window)
                    if tok0 < lo:
                        assert 0 < min(lo - tok0, TILE) <= TILE         # rows in front of the window
                    for rows in (4, 8):
                        shift = rows.bit_length() - 1
                        boxes = max(0, min(TILE, second_read - tok0 + rows - 1)) >> shift
                        first_box = max(0, lo - tok0) >> shift
                        assert 0 <= boxes - first_box <= TILE // rows
