"""Sizes of 8-bit projections that together take every way through the kernels: (m, n, k, gated).  The tiled form's ring
takes two blocks of 64 columns or more; from 8 on its loop runs, four blocks at a time, and 4 or 6 are left for its last
stages.  Single rows: each number of units that a thread holds, of one row and of several, and a wavefront's weights past
the first ones in flight."""

# m, n for each shape of the tiled form: 8 x 8, 14 x 16, 16 x 14 and 16 x 16 tiles
TILED = {False: {0: (1000, 2050), 1: (900, 14300), 2: (1800, 5000), 3: (4000, 4090)},
         True: {0: (1100, 1600), 2: (1800, 5000), 3: (900, 7200)}}
# blocks -> k, the last block partly or wholly behind the last column
COLUMNS = {2: 100, 4: 200, 6: 384, 8: 385, 10: 600, 12: 768, 14: 890, 64: 4096}

TILE_CASES = [(m, n, k, gated) for gated in (False, True) for m, n in TILED[gated].values() for k in COLUMNS.values()]

ROW_CASES = [(m, n, k, gated) for gated in (False, True) for m, n, k in [
    (1, 60, 2400), (1, 90, 4096), (1, 40, 4097), (1, 40, 8192), (1, 33, 8193), (1, 40, 16383), (1, 40, 16384),
    (2, 50, 4096), (2, 40, 4097), (2, 33, 8192), (3, 40, 4096), (4, 70, 4095), (4, 33, 4096),
    (1, 14336, 4096), (1, 32000, 2048), (3, 33000, 1100), (1, 33000, 1100)]]
# just past what a thread holds: rows are quantized by a kernel of their own
PAST_ROWS = [(m, n, k, gated) for gated in (False, True) for m, n, k in [
    (1, 40, 16385), (2, 40, 8193), (3, 40, 4097), (4, 40, 4097)]]
