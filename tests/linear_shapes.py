"""Shapes that reach every kernel of the 16-bit and 4-bit products, unsplit and split along K wherever their plans split them,
and products in parts along rows and columns. Ragged: rows, columns and K end inside a tile, a stage and a piece of 16 bytes."""

KERNELS = ["tile 256x256", "tile 256x128", "tile 128x128", "int4 256x256", "int4 128x256", "few 16 1/16/1", "few 16 1/8/2",
           "few 16 2/8/1", "few 16 2/4/2", "few 16 2/16/1", "few 32 1/4/4", "few 32 2/4/4", "few 32 2/4/2", "few 32 4/4/2",
           "few 64 2/4/2"]

# Of a kind of product: (rows, outputs, K) -> its launches, each a kernel and whether K is split.
PRODUCT = {
    (1, 33, 40): [("tile 128x128", False)],
    (3, 35, 1037): [("tile 128x128", True)],
    (1211, 11743, 713): [("tile 256x256", False)],
    (149, 16429, 6825): [("tile 256x256", True)],
    (385, 15241, 2507): [("tile 256x128", False)],
    (391, 7789, 6847): [("tile 256x128", True)],
    (443, 16453, 2143): [("tile 256x128", False), ("tile 128x128", True)],
    (921, 17313, 1803): [("tile 256x256", False), ("tile 128x128", True)],
    (1025, 21903, 3585): [("tile 256x256", False), ("tile 128x128", False), ("tile 128x128", True)],
}
GATED = {
    (1, 33, 40): [("few 16 2/8/1", False)],
    (3, 35, 4104): [("few 16 2/8/1", True)],
    (3, 4203, 8200): [("few 16 2/4/2", False)],
    (5, 45, 8200): [("few 16 2/4/2", True)],
    (19, 10301, 72): [("few 32 4/4/2", False)],
    (17, 33, 136): [("few 32 2/4/2", False)],
    (23, 45, 2056): [("few 32 2/4/2", True)],
    (39, 33, 520): [("few 64 2/4/2", False)],
    (61, 45, 2056): [("few 64 2/4/2", True)],
    (65, 33, 40): [("tile 128x128", False)],
    (67, 45, 1032): [("tile 128x128", True)],
    (139, 21571, 1224): [("tile 256x256", False)],
    (409, 4935, 6032): [("tile 256x256", True)],
    (65, 15629, 2008): [("tile 256x128", False)],
    (129, 6253, 11104): [("tile 256x128", True)],
    (1343, 3171, 1968): [("tile 128x128", False), ("few 64 2/4/2", True)],
    (1027, 4057, 2120): [("tile 256x128", False), ("few 16 2/8/1", False)],
    (683, 11067, 1200): [("tile 256x256", False), ("tile 128x128", True)],
    (1281, 8931, 1152): [("tile 256x256", False), ("tile 128x128", False), ("few 16 2/8/1", False)],
}
INT4 = {
    (1, 33, 39): [("few 16 1/16/1", False)],
    (3, 35, 16389): [("few 16 1/16/1", True)],
    (9, 4203, 71): [("few 16 1/8/2", False)],
    (11, 8301, 133): [("few 16 2/8/1", False)],
    (17, 33, 135): [("few 32 1/4/4", False)],
    (23, 45, 2055): [("few 32 1/4/4", True)],
    (39, 33, 519): [("few 64 2/4/2", False)],
    (61, 45, 2055): [("few 64 2/4/2", True)],
    (65, 33, 39): [("int4 128x256", False)],
    (67, 45, 1031): [("int4 128x256", True)],
    (71, 35, 1977): [("few 64 2/4/2", True), ("few 16 1/16/1", False)],
    (911, 15747, 709): [("int4 256x256", False)],
    (129, 20637, 4239): [("int4 256x256", True)],
    (987, 16793, 1095): [("int4 256x256", False), ("int4 128x256", True)],
    (261, 10293, 2257): [("int4 128x256", True), ("few 16 2/8/1", False)],
    (1297, 13749, 1909): [("int4 256x256", False), ("int4 128x256", True), ("few 32 1/4/4", False)],
}
INT4_GATED = {
    (1, 33, 39): [("few 16 2/8/1", False)],
    (3, 35, 8190): [("few 16 2/8/1", True)],
    (3, 35, 8197): [("few 16 2/16/1", False)],
    (5, 35, 16389): [("few 16 2/16/1", True)],
    (9, 8301, 71): [("few 16 2/4/2", False)],
    (19, 10301, 71): [("few 32 2/4/4", False)],
    (17, 33, 135): [("few 32 2/4/2", False)],
    (23, 45, 2055): [("few 32 2/4/2", True)],
    (39, 33, 519): [("few 64 2/4/2", False)],
    (61, 45, 2055): [("few 64 2/4/2", True)],
    (65, 33, 39): [("int4 128x256", False)],
    (67, 45, 1031): [("int4 128x256", True)],
    (107, 45, 7705): [("few 64 2/4/2", True), ("few 64 2/4/2", True)],
    (423, 16075, 665): [("int4 256x256", False)],
    (129, 10035, 4777): [("int4 256x256", True)],
    (509, 16779, 1343): [("int4 256x256", False), ("int4 128x256", True)],
    (799, 3547, 4267): [("int4 256x256", True), ("few 32 2/4/2", True)],
}
# Which of the kernels have no K split in any plan.
NEVER_SPLIT = {"few 16 1/8/2", "few 32 4/4/2", "few 32 2/4/4"}
