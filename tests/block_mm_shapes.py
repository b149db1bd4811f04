"""Shapes (rows, columns, K) that reach every kernel of the block-scaled product, unsplit and split along K wherever its plan
splits it, and products cut along rows and columns. Ragged everywhere: K ends inside a block and inside a 16-byte piece, and
gives a workgroup more blocks than it has in flight, so that every slot and register is used again."""

KERNELS = ["tile 64x64", "tile 64x128", "tile 128x128", "tile 128x256", "tile 256x128", "tile 256x256", "stream 1x1",
           "stream 1x1 wide", "stream 1x4", "stream 2x1", "stream 2x4", "stream 4x1"]

# shape -> its launches: (kernel, whether K is split)
LAUNCHES = {
    (1, 390, 3501): [("stream 1x1", False)],
    (1, 20, 14341): [("stream 1x1", True)],
    (1, 4083, 7003): [("stream 1x1 wide", False)],
    (16, 8203, 3003): [("stream 1x4", False)],
    (9, 4100, 8203): [("stream 1x4", True)],
    (23, 2100, 3003): [("stream 2x1", False)],
    (17, 20, 10005): [("stream 2x1", True)],
    (24, 8203, 3003): [("stream 2x4", False)],
    (24, 4100, 10011): [("stream 2x4", True)],
    (47, 120, 1003): [("stream 4x1", False)],
    (64, 100, 10011): [("stream 4x1", True)],
    (65, 130, 1003): [("tile 64x64", False)],
    (72, 17, 4003): [("tile 64x64", True)],
    (131, 5595, 1053): [("tile 64x128", False)],
    (65, 4167, 1826): [("tile 64x128", True)],
    (5573, 261, 1003): [("tile 128x128", False)],
    (257, 3323, 2729): [("tile 128x128", True)],
    (1312, 5426, 1031): [("tile 128x256", False)],
    (263, 7081, 4821): [("tile 128x256", True)],
    (5551, 646, 1004): [("tile 256x128", False)],
    (3452, 568, 3829): [("tile 256x128", True)],
    (1411, 5383, 1002): [("tile 256x256", False)],
    (3765, 2800, 5637): [("tile 256x256", True)],
    # cut: along columns, along rows, along both
    (4097, 5000, 2570): [("tile 256x256", False), ("tile 256x128", False)],
    (4984, 4619, 1060): [("tile 256x256", False), ("tile 128x256", False)],
    (4637, 5074, 1561): [("tile 256x256", False), ("tile 256x128", False), ("stream 2x1", False)],
}
# one row is split over 16 waves only where its columns fill the chip, and then not over workgroups
NEVER_SPLIT = {"stream 1x1 wide"}
# blocks of 128 that a workgroup has in flight: its ring's slots, or two (wide columns: one) for each of its waves
IN_FLIGHT = dict(zip(KERNELS, (4, 3, 3, 3, 3, 2, 16, 32, 8, 16, 16, 16)))
# beside few columns a longer K is split at once
NEVER_LONG = {("stream 4x1", False)}
